// Attention over an 8-bit paged cache (kv_pages.h): codes go from memory to
// the matrix cores as they are stored, never widened.
//
//   o[q] = sum_k w[k] v[k] / sum_k w[k],  w[k] = exp(sm_scale * q.k) over the keys q sees
//
// The matrix cores multiply e4m3 by e4m3 only, at twice the bf16 rate, so the
// bf16 side of each product is split: a bf16 value (8 significant bits) is the
// sum of two e4m3 values (4 bits each, signed remainder), an fp16 value (11) of
// three, each term 32 times finer than the one before.  Two terms cost what one
// bf16 product would, and K and V are neither converted nor read wider.
//   S^T = K Q^T   K rows are operand A as stored; q's terms operand B
//   O^T = V^T P^T V is stored [dim][token]: again operand A as stored; P's terms
//                 come from the S^T accumulators in the lane that holds them: the
//                 key order of S^T's rows is chosen so that a lane's accumulators are
//                 its P operand in V's token order.
// Powers of two are the instruction's own scale operands: a page's K and V
// scales, a query's scale, and, for P, the softmax's reference.  Weights are
// w = 2^(x - E + 8), x the logit in log2 units and E the least integer above the row's
// largest x among the keys at hand, so w lies in (0, 256] whatever its row's running
// maximum is; their operand's scale is 2^(E - 8 - M).  M, the row's reference,
// may therefore be any power of two near the maximum: it moves only when E exceeds
// it by 64, which rescales O and the sum exactly and happens at a row's first keys
// and hardly ever again.  While M stays, O and the sum may grow by 2^64:
// finite results take values below 2^63 over the number of keys.
//
// Precision.  Remainders keep w's error below 2^-8 (bf16) or 2^-12 (fp16) of itself, or
// 2^-22 of the largest; its sum is fp32, of w (bf16: rounded to fp16, 11 bits, which the
// terms come by too).  Accumulators are fp32, but the instructions align a sum's products
// before they add them: it is off by up to 2^-12 of the sum of their magnitudes (measured on
// codes of any exponents 2.0e-4 at worst and 2.9e-5 in the mean square, on Gaussian q and K
// 2.9e-5 and 2.8e-6).  A logit is off by as much of sm_scale * sum |q k|, and its weight by
// that part of itself.
//
// Three kernels.  attend_few: up to 16 (query, head) rows of one key/value head
// per workgroup, bound by the cache's bytes: 16x16x128 products, K and V loaded
// straight into operand registers, pages shared out over waves and workgroups.
// attend_some: the same for up to 32 rows, 32x32x64 products on half pages.
// attend_tile: 128 rows, 32 a wave, bound by products and exponentials: 32x32x64
// products from a double-buffered LDS stage.  Each splits a long axis over
// workgroups where rows alone leave CUs idle; join_few and join_tile add the pieces.
//
// Measured, 32 query and 8 key/value heads of 128: one token for each of 128 ragged
// sequences of up to 16000 tokens 365 us (5.4 TB/s; 5.1 is a copy's rate), for one
// sequence of 262000 97 us (5.5); 5 for each of 16 of 6000 47 us (4.2).  8448 rows over
// 25344 tokens x 12 heads 1.10 to 1.17 ms: 1.12 to 1.19 PFLOP/s, where an 8192^3 bf16 product
// reaches 1.21; the clock falls to 1.9 GHz, at which the vector units are busy for 70
// % of the time and the matrix cores for 53.  The same in fp16 1.60 ms (three terms are one and a
// half fp16 products, and more vector work), with 24 heads of 64 1.55 ms (the softmax's work for
// half the products).
#include <algorithm>
#include <type_traits>

#include "attn_terms.h"

namespace {

struct Args {
  fvsr_kv_cache c;
  const uint16_t* q;
  uint16_t* out;
  int64_t q_ts, q_hs, o_ts, o_hs;
  const uint8_t* keep;
  int64_t keep_q, keep_k;
  float* part;       // splits > 1: O of each row of each piece, then (M, l)
  float scale_log2;  // sm_scale * log2(e)
  int T, q_heads, group, causal, splits, tiles, tail;
  int whole, pieces;  // attend_tile: units done by one workgroup; workgroups of a later one
  int tile_rows;      // rows of a tile at most
};

// Keys that row i of a sequence sees.
FVSR_DEV int row_limit(const Args& a, const SeqPart& s, int i) {
  const int64_t cap = a.c.table_pages * kPage;
  const int lim = a.causal ? min(s.len, s.len - s.rows.n + i + 1) : s.len;
  return (int)min((int64_t)max(lim, 0), cap);
}

// The tile-th of all sequences' tiles of ROWS rows, n * pack rows to a sequence.
template <int ROWS>
FVSR_DEV bool tile_of(const Args& a, int tile, int pack, SeqPart& s) {
  const auto tiles_of = [pack](int n, int) { return (n * pack + ROWS - 1) / ROWS; };
  if (a.c.cu)
    return find_part(a.c.cu, a.c.lengths, (int)a.c.sequences, a.T, tile, a.tail != 0, tiles_of, s);
  const int each = a.tiles / (int)a.c.sequences;
  s.b = tile / each;
  s.part = tile % each;
  s.rows = seq_rows(nullptr, s.b, (int)a.c.sequences, a.T);
  s.len = max(a.c.lengths[s.b], 0);
  return true;
}

// A workgroup's unit of few rows: ROWS rows of a sequence, a head and a share of the
// pages.
struct FewUnit {
  SeqPart s;
  int split, h, rows, row0;  // rows: of the sequence; row0: the unit's first
};
template <int ROWS>
FVSR_DEV bool few_unit(const Args& a, FewUnit& u) {
  if (ROWS == 32 || !a.c.cu) {  // one unit to a sequence and head
    u.split = blockIdx.x, u.h = blockIdx.y;
    u.s.b = blockIdx.z, u.s.part = 0;
    u.s.rows = seq_rows(nullptr, u.s.b, (int)a.c.sequences, a.T);
    u.s.len = max(a.c.lengths[u.s.b], 0);
  } else {
    // The units of one sequence, head and split are neighbours on one XCD, which
    // read the same pages.
    const int at = xcd_order(blockIdx.x, gridDim.x);
    u.split = at / a.tiles % a.splits, u.h = at / a.tiles / a.splits;
    if (!tile_of<ROWS>(a, at % a.tiles, a.group, u.s)) return false;
  }
  u.rows = u.s.rows.n * a.group, u.row0 = u.s.part * ROWS;
  return true;
}

// Adds the waves' parts of each row (O at lds_o[wave][row], P floats apart; M and l in
// lds_ml) and writes the output, or the piece of it that join_few adds.
template <int DT, int D, int ROWS, int P>
FVSR_DEV void finish_few(const Args& a, const FewUnit& u, const float* lds_o,
                         const float (&lds_ml)[4][ROWS][2]) {
  __syncthreads();
  constexpr int C = D / 8;  // threads of a row
  const int d0 = threadIdx.x % C * 8;
  for (int i = threadIdx.x / C; i < ROWS && u.row0 + i < u.rows; i += kThreads / C) {
    const int row = u.row0 + i;
    float top = lds_ml[0][i][0];
#pragma unroll
    for (int w = 1; w < 4; ++w) top = fmaxf(top, lds_ml[w][i][0]);
    float o[8] = {}, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = __builtin_amdgcn_exp2f(lds_ml[w][i][0] - top);
      sum += f * lds_ml[w][i][1];
      const v4f x = *(const v4f*)&lds_o[(w * ROWS + i) * P + d0];
      const v4f y = *(const v4f*)&lds_o[(w * ROWS + i) * P + d0 + 4];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += f * x[e], o[4 + e] += f * y[e];
    }
    const int64_t token = u.s.rows.lo + row / a.group;
    const int oh = u.h * a.group + row % a.group;
    if (a.splits == 1) {
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      u32x2_t* op = (u32x2_t*)(a.out + token * a.o_ts + oh * a.o_hs + d0);
      op[0] = u32x2_t{pack2<DT>(o[0] * inv, o[1] * inv), pack2<DT>(o[2] * inv, o[3] * inv)};
      op[1] = u32x2_t{pack2<DT>(o[4] * inv, o[5] * inv), pack2<DT>(o[6] * inv, o[7] * inv)};
    } else {
      const int64_t pr = (token * a.q_heads + oh) * a.splits + u.split;
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

// ---------------------------------------------------------------------------
// attend_few.  Operand layout of v_mfma_scale_f32_16x16x128: lane (r, g) = (l %
// 16, l / 16) holds positions 16 g .. and 64 + 16 g .. (16 each) of row r; the
// scale of 32 positions 32 j .. of row r comes from lane (r, j); accumulator j
// of lane (q, g) is row 4 g + j of column q.
// ---------------------------------------------------------------------------
template <int DT, int D>
__global__ __launch_bounds__(kThreads, 2) void attend_few(Args a) {
  constexpr int N = terms(DT);
  constexpr int W = D / 64;                    // 16-byte pieces of a K row per lane
  constexpr int F = D == 128 ? N : (N + 1) / 2;  // Q operands (64 dims: two terms each)
  constexpr int DT16 = D / 16;
  constexpr int P = D + 4;
  __shared__ __attribute__((aligned(16))) float lds_o[4 * 16 * P];
  __shared__ float lds_ml[4][16][2];
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int H = (int)a.c.heads;
  FewUnit u;
  if (!few_unit<16>(a, u)) return;
  const SeqPart& s = u.s;
  const int h = u.h, rows = u.rows, row0 = u.row0, row1 = min(row0 + 16, rows);
  const int r = min(row0 + col, rows - 1);
  const int qi = r / a.group, hq = h * a.group + r % a.group;
  const int limit = row_limit(a, s, qi);
  const int lim_lo = row_limit(a, s, row0 / a.group);
  const int lim_hi = row_limit(a, s, (row1 - 1) / a.group);
  const int pages = (lim_hi + kPage - 1) / kPage;
  const int p0 = range_at(pages, u.split, a.splits), p1 = range_at(pages, u.split + 1, a.splits);
  const int32_t* const table = a.c.table + s.b * a.c.table_stride;

  // Q^T's terms.
  v8i qf[F];
  int qs[F];
  {
    const uint16_t* qp = a.q + (int64_t)(s.rows.lo + qi) * a.q_ts + (int64_t)hq * a.q_hs + 16 * g;
    u32x4_t raw[W][2];
#pragma unroll
    for (int w = 0; w < W; ++w) {
      raw[w][0] = *(const u32x4_t*)(qp + 64 * w);
      raw[w][1] = *(const u32x4_t*)(qp + 64 * w + 8);
    }
    const auto el = [&](int w, int i) {
      const uint32_t u = raw[w][i >> 3][(i >> 1) & 3];
      return to_f<DT>((uint16_t)(i & 1 ? u >> 16 : u & 0xffff));
    };
    uint32_t top = 0;
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = max_mag(top, el(w, i));
    top = max(top, (uint32_t)__shfl_xor((int)top, 16));
    top = max(top, (uint32_t)__shfl_xor((int)top, 32));
    const int e = row_exp(top);
    const float f = __builtin_ldexpf(1.0f, -e);
    uint32_t t[W][4][N];
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        split4<N>(el(w, 4 * i) * f, el(w, 4 * i + 1) * f, el(w, 4 * i + 2) * f,
                  el(w, 4 * i + 3) * f, t[w][i]);
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
  }

  v4f acc[DT16] = {};
  float m = kNothing, l = 0.0f;
  // Row r of K subtile t is key 64 (t / 4) + 16 (r / 4) + 4 (t % 4) + r % 4, so
  // that accumulator (t, j) of lane g is position 64 (t / 4) + 16 g + 4 (t % 4) + j.
  const int k_off = (16 * (col >> 2) + (col & 3)) * D + 16 * g;
  const int v_off = col * kPage + 16 * g;
  int ahead = p0 + wave < p1 ? table[p0 + wave] : 0;
  for (int p = p0 + wave; p < p1; p += 4) {
    const int64_t id = __builtin_amdgcn_readfirstlane(ahead);
    if (p + 4 < p1) ahead = table[p + 4];
    if (id < 0 || id >= a.c.pages) {  // no such page: the rows that would read it are NaN
      if (p * kPage < limit) l = __builtin_nanf("");
      continue;
    }
    const int64_t ph = id * H + h;
    const uint8_t* kp = (const uint8_t*)a.c.k + ph * kPage * D + k_off;
    const uint8_t* vp = (const uint8_t*)a.c.v + ph * kPage * D + v_off;
    const int ks = ((const uint8_t*)a.c.k_scale)[ph];
    int vs = ((const uint8_t*)a.c.v_scale)[ph];
    v8i kf[8], vf[DT16];
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const uint8_t* x = kp + ((t >> 2) * 64 + (t & 3) * 4) * D;
      const u32x4_t u = *(const u32x4_t*)x;
      kf[t] = join(u, D == 128 ? *(const u32x4_t*)(x + 64) : u);
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
      sc[t] = mfma(kf[t], qf[0], z, ks, qs[0]);
#pragma unroll
      for (int k = 1; k < F; ++k) sc[t] = mfma(kf[t], qf[k], sc[t], ks, qs[k]);
    }
    const bool masked = (p + 1) * kPage > lim_lo;
    if (masked) {
      const int at = p * kPage + 16 * g;
#pragma unroll
      for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (at + (t >> 2) * 64 + (t & 3) * 4 + j >= limit) sc[t][j] = -__builtin_huge_valf();
    }
    float top = -__builtin_huge_valf();
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) top = fmaxf(top, sc[t][j]);
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    int shift;
    weigh(sc, top, a.scale_log2, m, l, shift, [&](float f) {
#pragma unroll
      for (int d = 0; d < DT16; ++d) acc[d] *= f;
    });
    v8i pf[N];
    float sum = 0.0f;
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      uint32_t w[N];
      weights4<N>(sc[t][0], sc[t][1], sc[t][2], sc[t][3], w, sum);
#pragma unroll
      for (int k = 0; k < N; ++k) pf[k][t] = (int)w[k];
    }
    l += __builtin_ldexpf(sum, shift);
    if (masked) {
      // Hidden tokens weigh 0, which a NaN code would not survive: NaN codes
      // leave the product and are counted for the rows that see them.  A NaN scale
      // stands for a page of them.
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
        v8i seen;
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          seen[t] = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (p * kPage + 16 * g + (t >> 2) * 64 + (t & 3) * 4 + j < limit)
              seen[t] |= 0x38 << (8 * j);
        }
#pragma unroll
        for (int d = 0; d < DT16; ++d) {
          const v8i ones = take_nan(vf[d]);
          const v4f z = {};
          const v4f n = mfma(ones, seen, z, 127, 127);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (n[j] > 0.0f) acc[d][j] = __builtin_nanf("");
        }
      }
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int ps = e8m0(shift - 5 * k);
#pragma unroll
      for (int d = 0; d < DT16; ++d) acc[d] = mfma(vf[d], pf[k], acc[d], vs, ps);
    }
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);

#pragma unroll
  for (int d = 0; d < DT16; ++d)
    *(v4f*)&lds_o[(wave * 16 + col) * P + d * 16 + 4 * g] = acc[d];
  if (g == 0) lds_ml[wave][col][0] = m, lds_ml[wave][col][1] = l;
  finish_few<DT, D, 16, P>(a, u, lds_o, lds_ml);
}

template <int DT, int D>
__global__ __launch_bounds__(kThreads) void join_few(Args a) {
  const int64_t row = blockIdx.x, rows = (int64_t)a.T * a.q_heads;
  // Rows behind the last sequence have pieces only where they are to be zeros.
  if (a.c.cu && !a.tail && row / a.q_heads >= a.c.cu[a.c.sequences]) return;
  join_row<DT, D>(a.part + row * a.splits * D, D,
                  a.part + rows * a.splits * D + row * a.splits * 2, 2, a.splits,
                  a.out + row / a.q_heads * a.o_ts + row % a.q_heads * a.o_hs);
}

// ---------------------------------------------------------------------------
// attend_tile.  v_mfma_scale_f32_32x32x64: lane (r, g) = (l % 32, l / 32) holds
// positions 16 g .. and 32 + 16 g .. of row r; accumulator 4 i + j of lane (q, g) is row
// 8 i + 4 g + j of column q.
// ---------------------------------------------------------------------------

// 16-byte pieces of a stage's rows are swapped about so that 16 lanes reading
// one piece of 16 of the rows above touch every bank once: the rows of a K
// operand differ in token bits 0, 1, 2 and 4 (128-byte rows: bit 0 is the bank
// half, 64-byte rows: bits 0-1 the quarter), those of a V operand in dim bits 0-3.
template <int D>
FVSR_DEV int k_swap(int key) {
  return D == 128 ? ((key >> 1) & 3) | ((key >> 2) & 4) : ((key >> 2) & 1) | ((key >> 3) & 2);
}
FVSR_DEV int v_swap(int d) { return (d >> 1) & 7; }

// A page's K or V codes go into LDS straight from memory, segment s (1 KB) by wave
// s % 4; the piece that a lane fetches is the one that belongs where it lands.  Offset of a
// lane's piece in its wave's first segment:
template <int D>
FVSR_DEV int k_piece(int wave, int lane) {
  constexpr int KR = D / 16;  // pieces of a row
  return wave * 1024 + lane / KR * D +
         ((lane % KR) ^ k_swap<D>(wave * (64 / KR) + lane / KR)) * 16;
}
FVSR_DEV int v_piece(int wave, int lane) {
  return wave * 1024 + lane / 8 * kPage + ((lane % 8) ^ v_swap(wave * 8 + lane / 8)) * 16;
}
template <int D>
FVSR_DEV void stream(uint8_t LDS_AS* to, const uint8_t* from, int wave, int& piece) {
  // (Opaque, so that no sum with it is kept in registers from page to page.)
  asm volatile("" : "+v"(piece));
#pragma unroll
  for (int t = 0; t < kPage * D / 4096; ++t)
    __builtin_amdgcn_global_load_lds(from + t * 4096 + piece,
                                     (void LDS_AS*)(to + wave * 1024 + t * 4096), 16, 0, 0);
}

// The pages ahead, looked up kList at a time: first position, id, K scale | V
// scale << 8.
constexpr int kList = 512;
typedef int v4i __attribute__((ext_vector_type(4)));
struct Listed {
  int n, whole;  // entries; those that every row of the tile sees whole (the first ones)
};

// Entries of pages from .. from + kList - 1 below p1 that the block mask's row
// keeps (null: all), in order.  A page id outside the pool has no entry: `bad` is the
// first position of any.  Every wave counts all pages and writes its share.
FVSR_DEV Listed list_pages(v4i LDS_AS* list, const Args& a, const int32_t* table, int h,
                           const uint8_t* keep, int kept, int from, int p1, int seen, int wave,
                           int& bad) {
  const int lane = threadIdx.x & 63;
  Listed c{0, 0};
#pragma unroll 1
  for (int g = 0; g < kList / 64 && from + g * 64 < p1; ++g) {
    const int i = from + g * 64 + lane;
    const bool in = i < p1 && (!keep || (i < kept && keep[i] != 0));
    const int id = in ? table[i] : 0;
    const bool there = in && id >= 0 && id < a.c.pages;
    const uint64_t word = __ballot(there), wrong = __ballot(in && !there);
    if (wrong) bad = min(bad, (from + g * 64 + __builtin_ctzll(wrong)) * kPage);
    if (there && g % 4 == wave) {
      const int64_t ph = (int64_t)id * a.c.heads + h;
      list[c.n + __popcll(word & ((1ull << lane) - 1))] =
          v4i{i * kPage, id,
              ((const uint8_t*)a.c.k_scale)[ph] | ((const uint8_t*)a.c.v_scale)[ph] << 8, 0};
    }
    c.n += __popcll(word);
    c.whole += __popcll(__ballot(there && (i + 1) * kPage <= seen));
  }
  return c;
}

// One wave's 32 rows.
//
// step(): pages that every row sees whole, in a pipeline of half pages (64 keys).
// Step t turns the logits S of half t into weights P while the matrix cores do O +=
// V P of half t - 1 and S of half t + 1, so that neither waits for the other even
// within a wave.  Its steps are one straight block, which is what lets the compiler
// keep to their order: the reference M stays that of the first half page, and a row that
// would have to move it is noted (`lost`).  The tile is then done again without the
// pipeline; it takes a logit 44 above all of that half page's.
// one(): any page, half by half, with masks, a moving M and NaN codes.
template <int DT, int D>
struct RowTile {
  static constexpr int N = terms(DT);
  v8i qf[D / 64][N];
  int qs[N];
  v16f acc[D / 32] = {};
  float m = kNothing, l = 0.0f;
  v8i pf[N];       // weights of the half before, and their scale
  int shift = 0;
  bool lost = false;
  int limit, lim_lo;  // keys this lane's row sees; least of the wave
  float c;
  int k_at[D / 32], v_at[2];  // this lane's pieces of an operand, half 0

  // Row r = 8 i + 4 g' + j of K subtile u is key 32 u + 16 g' + 4 i + j.
  static __device__ __forceinline__ int k_row(int r) {
    return 16 * ((r >> 2) & 1) + 4 * (r >> 3) + (r & 3);
  }
  // The terms of this lane's row.
  __device__ __forceinline__ void load_q(const uint16_t* row) {
    const uint16_t* qp = row + 16 * ((threadIdx.x >> 5) & 1);
    u32x4_t raw[D / 32][2];
#pragma unroll
    for (int x = 0; x < D / 32; ++x) {
      raw[x][0] = *(const u32x4_t*)(qp + 32 * x);
      raw[x][1] = *(const u32x4_t*)(qp + 32 * x + 8);
    }
    const auto el = [&](int x, int i) {
      const uint32_t u = raw[x][i >> 3][(i >> 1) & 3];
      return to_f<DT>((uint16_t)(i & 1 ? u >> 16 : u & 0xffff));
    };
    uint32_t top = 0;
#pragma unroll
    for (int x = 0; x < D / 32; ++x)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = max_mag(top, el(x, i));
    top = max(top, (uint32_t)__shfl_xor((int)top, 32));
    const int e = row_exp(top);
    const float f = __builtin_ldexpf(1.0f, -e);
#pragma unroll
    for (int k = 0; k < N; ++k) qs[k] = e8m0(e - 5 * k);
#pragma unroll
    for (int x = 0; x < D / 32; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t t[N];
        split4<N>(el(x, 4 * i) * f, el(x, 4 * i + 1) * f, el(x, 4 * i + 2) * f,
                  el(x, 4 * i + 3) * f, t);
#pragma unroll
        for (int k = 0; k < N; ++k) qf[x >> 1][k][(x & 1) * 4 + i] = (int)t[k];
      }
  }
  __device__ __forceinline__ void place() {
    const int lane = threadIdx.x & 63, r = lane & 31, g = lane >> 5;
    const int kr = k_row(r);
#pragma unroll
    for (int w = 0; w < D / 32; ++w) k_at[w] = kr * D + (((2 * w + g) ^ k_swap<D>(kr)) << 4);
#pragma unroll
    for (int w = 0; w < 2; ++w) v_at[w] = r * kPage + (((2 * w + g) ^ v_swap(r)) << 4);
  }
  // Makes the addresses unknown, as in stream().
  __device__ __forceinline__ void fresh() {
#pragma unroll
    for (int w = 0; w < D / 32; ++w) asm volatile("" : "+v"(k_at[w]));
    asm volatile("" : "+v"(v_at[0]), "+v"(v_at[1]));
  }
  __device__ __forceinline__ v8i k_operand(const uint8_t LDS_AS* k, int half, int u, int w) const {
    const uint8_t LDS_AS* p = k + (half * 64 + u * 32) * D;
    return join(*(const u32x4_t LDS_AS*)(p + k_at[2 * w]),
                *(const u32x4_t LDS_AS*)(p + k_at[2 * w + 1]));
  }
  __device__ __forceinline__ v8i v_operand(const uint8_t LDS_AS* v, int half, int d) const {
    const uint8_t LDS_AS* p = v + d * 32 * kPage;  // (half 1: piece ^ 4)
    return join(*(const u32x4_t LDS_AS*)(p + (v_at[0] ^ (half * 64))),
                *(const u32x4_t LDS_AS*)(p + (v_at[1] ^ (half * 64))));
  }
  // (k_of(u, w): the K operand of 32 keys u and 64 dims w of the half.)
  template <class K>
  __device__ __forceinline__ void logits(v16f (&s)[2], K k_of, int ks) {
#pragma unroll
    for (int u = 0; u < 2; ++u) s[u] = v16f{};
#pragma unroll
    for (int w = 0; w < D / 64; ++w)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const v8i kf = k_of(u, w);
#pragma unroll
        for (int t = 0; t < N; ++t) s[u] = mfma(kf, qf[w][t], s[u], ks, qs[t]);
      }
  }
  __device__ __forceinline__ void add_values(const uint8_t LDS_AS* v, int half, int vs) {
#pragma unroll
    for (int d = 0; d < D / 32; ++d) {
      const v8i vf = v_operand(v, half, d);
#pragma unroll
      for (int t = 0; t < N; ++t) acc[d] = mfma(vf, pf[t], acc[d], vs, e8m0(shift - 5 * t));
    }
  }
  // The order of a phase with n products: after each its share of exponentials
  // and of other arithmetic; two LDS reads before each operand's first product.
  template <bool EXP, bool MFMA, int TRANS, int VALU>
  static __device__ __forceinline__ void order(int n) {
#pragma unroll
    for (int i = 0; i < n; ++i) {
      if (MFMA) {
        if (i % N == 0) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      }
      if (EXP) __builtin_amdgcn_sched_group_barrier(0x400, TRANS, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, VALU, 0);
    }
  }
  static __device__ __forceinline__ float top_of(const v16f (&s)[2]) {
    float top = -__builtin_huge_valf();
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, s[u][e]);
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top),
                                                     false, false);
    return fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
  }
  // E of the logits at hand.
  __device__ __forceinline__ float exponent(const v16f (&s)[2]) const {
    return fmaxf(__builtin_ceilf(top_of(s) * c), kNothing);
  }
  // Step of the half whose logits are s: PV: with the half before (its V in v,
  // half pv_half), QK: with the logits of the half behind (into next).
  template <bool PV, bool QK>
  __device__ __forceinline__ void step(v16f (&s)[2], v16f (&next)[2], const uint8_t LDS_AS* v,
                                       int pv_half, int vs, const uint8_t LDS_AS* k, int qk_half,
                                       int ks) {
    const float e = exponent(s);
    lost |= e > m + 64.0f;
    // Each product is followed by its share of the arithmetic, which it runs
    // beside; operands are read from LDS one product ahead.
    const float off = 8.0f - e;
    v8i f{}, ahead{};
    constexpr int P1 = D / 32 * N;  // products of O
    if constexpr (PV) ahead = v_operand(v, pv_half, 0);
#pragma unroll
    for (int i = 0; i < P1; ++i) {
      const int d = i / N, t = i % N;
      if (t == 0) {
        f = ahead;
        if (d + 1 < D / 32) {
          if constexpr (PV) ahead = v_operand(v, pv_half, d + 1);
        } else {
          if constexpr (QK) ahead = k_operand(k, qk_half, 0, 0);
        }
      }
      if constexpr (PV) acc[d] = mfma(f, pf[t], acc[d], vs, e8m0(shift - 5 * t));
#pragma unroll
      for (int x = 32 * i / P1; x < 32 * (i + 1) / P1; ++x)
        s[x >> 4][x & 15] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x >> 4][x & 15], c, off));
    }
    order<true, PV, (32 + P1 - 1) / P1, (32 + P1 - 1) / P1 + 1>(P1);
    __builtin_amdgcn_sched_barrier(0);
    shift = (int)fmaxf(e - m, -300.0f) - 8;
    float sum = 0.0f;
    constexpr int P2 = D / 64 * 2 * N;  // products of the next S
    if constexpr (QK) next[0] = next[1] = v16f{};
#pragma unroll
    for (int i = 0; i < P2; ++i) {
      const int x = i / N, t = i % N, u = x & 1, w = x >> 1;
      if constexpr (QK) {
        if (t == 0) {
          f = ahead;
          if (x + 1 < P2 / N) ahead = k_operand(k, qk_half, (x + 1) & 1, (x + 1) >> 1);
        }
        next[u] = mfma(f, qf[w][t], next[u], ks, qs[t]);
      }
#pragma unroll
      for (int g = 8 * i / P2; g < 8 * (i + 1) / P2; ++g) {
        uint32_t o[N];
        const v16f& sg = s[g >> 2];
        const int b = 4 * (g & 3);
        weights4<N>(sg[b], sg[b + 1], sg[b + 2], sg[b + 3], o, sum);
#pragma unroll
        for (int n = 0; n < N; ++n) pf[n][g] = (int)o[n];
      }
    }
    l += __builtin_ldexpf(sum, shift);
    order<false, QK, 0, (8 * (N == 2 ? 12 : 22) + P2 - 1) / P2>(P2);
    __builtin_amdgcn_sched_barrier(0);
  }
  // A half page at position `at`, v_of(d) being the V operand of 32 dims: any, with masks, a
  // moving M and NaN codes.  after() runs once K is no longer needed.
  template <class K, class V, class After>
  __device__ __forceinline__ void half_page(K k_of, V v_of, int at, int ks, int vs, After after) {
    v16f s[2];
    logits(s, k_of, ks);
    after();
    const int room = limit - at - 16 * ((threadIdx.x >> 5) & 1);  // 32 u + e < it
    const bool masked = at + 64 > lim_lo;
    if (masked) {
      asm volatile("" :::);  // a branch: most pages are seen whole
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (32 * u + e >= room) s[u][e] = -__builtin_huge_valf();
    }
    weigh(s, top_of(s), c, m, l, shift, [&](float f) {
#pragma unroll
      for (int d = 0; d < D / 32; ++d) acc[d] *= f;
    });
    float sum = 0.0f;
#pragma unroll
    for (int g = 0; g < 8; ++g) {
      uint32_t o[N];
      const v16f& sg = s[g >> 2];
      const int b = 4 * (g & 3);
      weights4<N>(sg[b], sg[b + 1], sg[b + 2], sg[b + 3], o, sum);
#pragma unroll
      for (int n = 0; n < N; ++n) pf[n][g] = (int)o[n];
    }
    l += __builtin_ldexpf(sum, shift);
    v8i seen{};  // 1.0 where this lane's row sees a token (masked halves)
    if (masked) {
      asm volatile("" :::);
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (32 * (i >> 2) + 4 * (i & 3) + j < room) seen[i] |= 0x38 << (8 * j);
    }
#pragma unroll
    for (int d = 0; d < D / 32; ++d) {
      v8i f = v_of(d);
      if (masked && (vs == 255 || __ballot(has_nan(f)) != 0)) {  // as in attend_few
        if (vs == 255) {
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = 0x7f7f7f7f;
        }
        const v8i ones = take_nan(f);
        const v16f z = {};
        const v16f n = mfma(ones, seen, z, 127, 127);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (n[e] > 0.0f) acc[d][e] = __builtin_nanf("");
      }
#pragma unroll
      for (int t = 0; t < N; ++t)
        acc[d] = mfma(f, pf[t], acc[d], masked && vs == 255 ? 127 : vs, e8m0(shift - 5 * t));
    }
  }
  // A page at position `at` in a stage.
  __device__ __forceinline__ void one(const uint8_t LDS_AS* k, const uint8_t LDS_AS* v, int at,
                                      int ks, int vs) {
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {
      fresh();
      half_page([&](int u, int w) { return k_operand(k, half, u, w); },
                [&](int d) { return v_operand(v, half, d); }, at + half * 64, ks, vs, [] {});
    }
  }
};

// attend_few for 17 to 32 rows: the same sharing out of pages, half a page at a time (a
// whole one's operands beside 32 rows' O are more than 256 registers).  The K operand of the
// half ahead loads as soon as the logits have used the one before it.  16 x 5 tokens x 32 / 8
// heads over 6000: 47 us (4.2 TB/s), by tiles of 128 rows 52.  Five tokens over 262000: 101 us (5.3
// TB/s), by tiles 108.
template <int DT, int D>
__global__ __launch_bounds__(kThreads, 2) void attend_some(Args a) {
  constexpr int P = D + 4;
  __shared__ __attribute__((aligned(16))) float lds_o[4 * 32 * P];
  __shared__ float lds_ml[4][32][2];
  const int lane = threadIdx.x & 63, r32 = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int H = (int)a.c.heads;
  FewUnit u;
  if (!few_unit<32>(a, u)) return;
  const SeqPart& s = u.s;
  const int row1 = min(u.row0 + 32, u.rows), r = min(u.row0 + r32, u.rows - 1);
  RowTile<DT, D> w;
  w.limit = row_limit(a, s, r / a.group);
  w.lim_lo = row_limit(a, s, u.row0 / a.group);
  w.c = a.scale_log2;
  const int last = row_limit(a, s, (row1 - 1) / a.group);
  const int pages = (last + kPage - 1) / kPage;
  const int p0 = range_at(pages, u.split, a.splits), p1 = range_at(pages, u.split + 1, a.splits);
  const int32_t* const table = a.c.table + s.b * a.c.table_stride;
  int look = p0 + wave, ahead = look < p1 ? table[look] : 0;
  w.load_q(a.q + (int64_t)(s.rows.lo + r / a.group) * a.q_ts +
           (int64_t)(u.h * a.group + r % a.group) * a.q_hs);
  // The wave's next page that exists (none: false); rows that would read others are NaN.
  int p = 0, ks = 0, vs = 0;
  const uint8_t *kp = nullptr, *vp = nullptr;
  const auto next = [&] {
    for (; look < p1; look += 4) {
      const int64_t id = __builtin_amdgcn_readfirstlane(ahead);
      if (look + 4 < p1) ahead = table[look + 4];
      if (id >= 0 && id < a.c.pages) {
        const int64_t ph = id * H + u.h;
        kp = (const uint8_t*)a.c.k + ph * kPage * D, vp = (const uint8_t*)a.c.v + ph * kPage * D;
        ks = ((const uint8_t*)a.c.k_scale)[ph], vs = ((const uint8_t*)a.c.v_scale)[ph];
        p = look;
        look += 4;
        return true;
      }
      if (look * kPage < w.limit) w.l = __builtin_nanf("");
    }
    return false;
  };
  const int k_off = RowTile<DT, D>::k_row(r32) * D + 16 * g, v_off = r32 * kPage + 16 * g;
  v8i kf[2][D / 64], vf[D / 32];
  const auto load_k = [&](const uint8_t* from) {
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int y = 0; y < D / 64; ++y) {
        const uint8_t* at = from + k_off + x * 32 * D + y * 64;
        kf[x][y] = join(*(const u32x4_t*)at, *(const u32x4_t*)(at + 32));
      }
  };
  bool more = next();
  if (more) load_k(kp);
#pragma unroll 1
  for (int half = 0; more;) {
    const int at = p * kPage + half * 64, k_scale = ks, v_scale = vs;
#pragma unroll
    for (int d = 0; d < D / 32; ++d) {
      const uint8_t* from = vp + v_off + d * 32 * kPage + half * 64;
      vf[d] = join(*(const u32x4_t*)from, *(const u32x4_t*)(from + 32));
    }
    if (half) more = next();
    half ^= 1;
    // (The last page's first half once more behind the last: no branch.)
    w.half_page([&](int x, int y) { return kf[x][y]; }, [&](int d) { return vf[d]; }, at, k_scale,
                v_scale, [&] { load_k(kp + half * 64 * D); });
  }
  const float l = w.l + __shfl_xor(w.l, 32);
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *(v4f*)&lds_o[(wave * 32 + r32) * P + d * 32 + 8 * i + 4 * g] =
          v4f{w.acc[d][4 * i], w.acc[d][4 * i + 1], w.acc[d][4 * i + 2], w.acc[d][4 * i + 3]};
  if (g == 0) lds_ml[wave][r32][0] = w.m, lds_ml[wave][r32][1] = l;
  finish_few<DT, D, 32, P>(a, u, lds_o, lds_ml);
}

// Unit u of a call: a head (of the queries with a block mask, else of the keys)
// and 128 rows of one sequence.  Without a mask a tile's rows are (query, head of the
// group) pairs, so a group's heads read its pages once; with one, each head has
// its own pages.
struct TileUnit {
  SeqPart s;
  int head, h, pack, rows;  // h: key/value head; rows: of the sequence
  __device__ __forceinline__ int query(int r) const { return r / pack; }
  __device__ __forceinline__ int q_head(const Args& a, int r) const {
    return a.keep ? head : h * a.group + r % pack;
  }
};
FVSR_DEV bool unit_of(const Args& a, int u, TileUnit& t) {
  t.pack = a.keep ? 1 : a.group;
  t.head = u / a.tiles;
  t.h = a.keep ? t.head / a.group : t.head;
  // Under a causal mask later tiles see more: they go first.
  if (!tile_of<128>(a, a.causal ? a.tiles - 1 - u % a.tiles : u % a.tiles, t.pack, t.s))
    return false;
  t.rows = t.s.rows.n * t.pack;
  return true;
}

template <int DT, int D>
__global__ __launch_bounds__(kThreads) void join_tile(Args a) {
  const int cut = blockIdx.x / a.tile_rows, r = blockIdx.x % a.tile_rows;
  const int64_t cuts = gridDim.x / a.tile_rows;
  TileUnit t;
  if (!unit_of(a, a.whole + cut, t)) return;
  const int row = t.s.part * 128 + r;
  if (row >= t.rows) return;
  const int64_t at = (int64_t)cut * a.pieces * 128 + r;
  join_row<DT, D>(a.part + at * D, 128 * D, a.part + cuts * a.pieces * 128 * D + at * 2, 128 * 2,
                  a.pieces,
                  a.out + (int64_t)(t.s.rows.lo + t.query(row)) * a.o_ts +
                      (int64_t)t.q_head(a, row) * a.o_hs);
}

template <int DT, int D>
__global__ __launch_bounds__(kThreads, 2) void attend_tile(Args a) {
  // Two pages' K and V: page i of the list in the even or odd ones.  Distinct
  // objects, so that the compiler can tell the loads into one from the reads of
  // another and does not wait for them.
  __shared__ __attribute__((aligned(1024))) uint8_t k_even[kPage * D], k_odd[kPage * D];
  __shared__ __attribute__((aligned(1024))) uint8_t v_even[kPage * D], v_odd[kPage * D];
  __shared__ v4i list[kList];
  __shared__ int again;
  uint8_t LDS_AS* const k0 = (uint8_t LDS_AS*)k_even;
  uint8_t LDS_AS* const k1 = (uint8_t LDS_AS*)k_odd;
  uint8_t LDS_AS* const v0 = (uint8_t LDS_AS*)v_even;
  uint8_t LDS_AS* const v1 = (uint8_t LDS_AS*)v_odd;
  const int lane = threadIdx.x & 63, r32 = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wg = blockIdx.x;
  const bool cut = wg >= a.whole;  // a piece of a unit
  const int cut_at = cut ? xcd_order(wg - a.whole, (int)gridDim.x - a.whole) : 0;
  const int piece = cut ? cut_at % a.pieces : 0, pieces = cut ? a.pieces : 1;
  TileUnit t;
  if (!unit_of(a, cut ? a.whole + cut_at / a.pieces : xcd_order(wg, a.whole), t)) return;
  const SeqPart& s = t.s;
  const int H = (int)a.c.heads, h = t.h, rows = t.rows;
  const int first = s.part * 128 + wave * 32;  // the wave's first row
  const int r = min(first + r32, rows - 1), qi = t.query(r), hq = t.q_head(a, r);
  RowTile<DT, D> w;
  w.limit = row_limit(a, s, qi);
  w.lim_lo = row_limit(a, s, t.query(min(first, rows - 1)));
  w.c = a.scale_log2;
  w.place();
  const int tile_lo = row_limit(a, s, t.query(s.part * 128));
  const int last = row_limit(a, s, t.query(min(s.part * 128 + 127, rows - 1)));
  const int pages = (last + kPage - 1) / kPage;
  const int32_t* const table = a.c.table + s.b * a.c.table_stride;
  const uint8_t* keep = nullptr;
  int kept = 0;
  if (a.keep) {
    keep = a.keep + (((int64_t)s.b * a.q_heads + t.head) * a.keep_q + s.part) * a.keep_k;
    kept = s.part < a.keep_q && s.b < a.c.sequences ? (int)min(a.keep_k, (int64_t)0x7fffffff) : 0;
  }
  const int p0 = range_at(pages, piece, pieces), p1 = range_at(pages, piece + 1, pieces);

  w.load_q(a.q + (int64_t)(s.rows.lo + qi) * a.q_ts + (int64_t)hq * a.q_hs);

  const uint8_t* const kb = (const uint8_t*)a.c.k + (int64_t)h * kPage * D;
  const uint8_t* const vb = (const uint8_t*)a.c.v + (int64_t)h * kPage * D;
  const int64_t stride = (int64_t)H * kPage * D;
  const auto entry = [&](int i) {
    v4i e = ((const v4i LDS_AS*)list)[i];
#pragma unroll
    for (int k = 0; k < 3; ++k) e[k] = __builtin_amdgcn_readfirstlane(e[k]);
    return e;
  };
  const auto wait_all = [] {
    __builtin_amdgcn_s_waitcnt(0);  // this wave's loads
    __syncthreads();                // ... and everyone's
  };
  int kp = k_piece<D>(wave, lane), vp = v_piece(wave, lane);
  int bad = 0x7fffffff;
  const auto k_of = [&](const v4i& e) { return kb + e[1] * stride; };
  const auto v_of = [&](const v4i& e) { return vb + e[1] * stride; };
  if (threadIdx.x == 0) again = 0;
  // A wave without rows (`live` false) only streams and waits with the others.
  const auto all_pages = [&](auto live) {
    for (bool piped = true;; piped = false) {
      for (int from = p0; from < p1; from += kList) {
        __syncthreads();
        const Listed c = list_pages((v4i LDS_AS*)list, a, table, h, keep, kept, from, p1, tile_lo,
                                    wave, bad);
        const int n = c.n;
        __syncthreads();
        if (n == 0) continue;
        v4i cur = entry(0), nxt = n > 1 ? entry(1) : cur;
        stream<D>(k0, k_of(cur), wave, kp);
        stream<D>(v0, v_of(cur), wave, vp);
        int i = 0;
        // The pipeline's pages: the first `e`, an odd number of them (a branch between
        // two pages makes the compiler spill).
        const int e = piped && c.whole > 2 ? (c.whole - 1) | 1 : 0;
        if (e > 0) {
          v16f sa[2], sb[2];
          // Page i's second half and the first of page i + 1.
          const auto pair = [&](uint8_t LDS_AS* k, uint8_t LDS_AS* v, uint8_t LDS_AS* k_next,
                                uint8_t LDS_AS* v_next) {
            wait_all();
            const v4i behind = entry(min(i + 2, n - 1));  // (the last one again: no branch)
            stream<D>(k, k_of(behind), wave, kp);
            stream<D>(v_next, v_of(nxt), wave, vp);
            if constexpr (live) {
              const int vs = cur[2] >> 8, ks = nxt[2] & 255;
              w.fresh();
              w.template step<true, true>(sb, sa, v, 0, vs, k_next, 0, ks);
              w.template step<true, true>(sa, sb, v, 1, vs, k_next, 1, ks);
            }
            cur = nxt;
            nxt = behind;
            ++i;
          };
          wait_all();
          stream<D>(k1, k_of(nxt), wave, kp);
          if constexpr (live) {
            w.logits(sa, [&](int u, int x) { return w.k_operand(k0, 0, u, x); }, cur[2] & 255);
            if (w.m == kNothing) w.m = w.exponent(sa);
            w.template step<false, true>(sa, sb, nullptr, 0, 0, k0, 1, cur[2] & 255);
          }
          while (i + 1 < e) {
            pair(k0, v0, k1, v1);
            pair(k1, v1, k0, v0);
          }
          wait_all();
          if (i + 1 < n) stream<D>(v1, v_of(nxt), wave, vp);
          if constexpr (live) {
            w.template step<true, false>(sb, sa, v0, 0, cur[2] >> 8, nullptr, 0, 0);
            w.add_values(v0, 1, cur[2] >> 8);
          }
          cur = nxt;
          ++i;
        }
        // Page i alone, its codes being on their way to k and v.
        const auto single = [&](uint8_t LDS_AS* k, uint8_t LDS_AS* v, uint8_t LDS_AS* k_next,
                                uint8_t LDS_AS* v_next) {
          wait_all();
          if (i + 1 < n) {
            nxt = entry(i + 1);
            stream<D>(k_next, k_of(nxt), wave, kp);
            stream<D>(v_next, v_of(nxt), wave, vp);
          }
          if constexpr (live) w.one(k, v, cur[0], cur[2] & 255, cur[2] >> 8);
          cur = nxt;
          ++i;
        };
        while (i < n) {
          if (!(i & 1)) single(k0, v0, k1, v1);
          if (i < n) single(k1, v1, k0, v0);
        }
      }
      if (!piped || p0 >= p1) break;
      if (__ballot(w.lost) != 0) again = 1;
      __syncthreads();
      if (!again) break;
#pragma unroll
      for (int d = 0; d < D / 32; ++d) w.acc[d] = v16f{};
      w.m = kNothing, w.l = 0.0f;
    }
  };
  if (first < rows)
    all_pages(std::true_type{});
  else
    all_pages(std::false_type{});

  float l = w.l + __shfl_xor(w.l, 32);
  if (w.limit > bad) l = __builtin_nanf("");  // the row reads a page that does not exist
  if (first + r32 >= rows) return;
  if (!cut) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint16_t* op = a.out + (int64_t)(s.rows.lo + qi) * a.o_ts + (int64_t)hq * a.o_hs + 4 * g;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *(u32x2_t*)(op + d * 32 + 8 * i) =
            u32x2_t{pack2<DT>(w.acc[d][4 * i] * inv, w.acc[d][4 * i + 1] * inv),
                    pack2<DT>(w.acc[d][4 * i + 2] * inv, w.acc[d][4 * i + 3] * inv)};
  } else {
    const int64_t total = (int64_t)((int)gridDim.x - a.whole);  // pieces of the call
    const int64_t at = (int64_t)cut_at * 128 + wave * 32 + r32;
    float* po = a.part + at * D + 4 * g;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *(v4f*)(po + d * 32 + 8 * i) =
            v4f{w.acc[d][4 * i], w.acc[d][4 * i + 1], w.acc[d][4 * i + 2], w.acc[d][4 * i + 3]};
    if (g == 0) {
      float* ml = a.part + total * 128 * D + at * 2;
      ml[0] = w.m, ml[1] = l;
    }
  }
}

// How a call is cut up: a function of its sizes (and the CUs) only.
struct Plan {
  int few;         // rows of a unit of attend_few (16) or attend_some (32); 0: attend_tile
  int64_t tiles;   // of 16 or 128 rows, per head, over all sequences
  int64_t units;   // tiles of all heads
  int64_t whole;   // units done by one workgroup each; the others by `pieces` each
  int pieces;
  int splits;      // attend_few: workgroups of a unit
  int64_t floats(int64_t T, int64_t q_heads, int64_t D) const {
    if (few) return splits > 1 ? T * q_heads * splits * (D + 2) : 0;
    return (units - whole) * pieces * 128 * (D + 2);
  }
};

Plan plan_attn(const fvsr_kv_cache* c, int64_t T, int64_t q_heads, bool keep) {
  Plan p{};
  const int64_t group = q_heads / c->heads, B = c->sequences, cus = cu_count();
  p.pieces = p.splits = 1;
  // Packed rows: at most this many tiles over any counts that add up to T, the
  // rows behind the last sequence included.
  const auto tiles = [&](int64_t pack, int64_t rows) {
    return c->cu ? T * pack / rows + B + 1 : B * ((T / B * pack + rows - 1) / rows);
  };
  // Rows of any number per sequence: where they are few on average, waiting for
  // memory is what counts, and 16 rows to a workgroup with its waves on pages of their own
  // wait less than 128 with one stream of pages, even if some units read the same pages.
  // (us in units of 16 / in tiles.  32 sequences of 1 to 16 tokens over up to 9000 x 32 / 8
  // heads 120 / 159, 16 of 1 to 32 over up to 9000 x 16 / 4 54 / 72, over up to 3000 25 / 42.  It
  // loses where lengths are short or one prompt holds most rows: 32 of 1 to 32 over up to 2000 x
  // 32 / 8 58 / 43, 128 single tokens over 3000 and a prompt of 1500 230 / 185.)  The same number
  // for each: if one unit of 16 or 32 holds them (20 rows over 6000 tokens: one of 32 47 us,
  // tiles 52) and a grid holds their heads and sequences.
  if (!keep && T * group <= B * (c->cu ? 64 : 32) &&
      (c->cu || (c->heads <= kMaxGridYZ && B <= kMaxGridYZ)))
    p.few = c->cu || T * group <= B * 16 ? 16 : 32;
  if (p.few) {
    p.tiles = tiles(group, p.few);
    p.units = p.tiles * c->heads;
    // Sequences may be of any lengths: 16 workgroups per CU even them out (128
    // ragged sequences of up to 16000 tokens, us at 4 / 8 / 16 / 32: 426, 376, 366, 373).
    // Two pages to a wave, or one where that would leave CUs idle (20000 tokens x 12
    // heads 17.9 us, 19.0 with one; 4 sequences of 5000 x 2 heads 14.3, 11.2 with one).
    // 32 rows cost more to write and to add again, so there it is one workgroup per CU (16
    // x 5 tokens x 32 / 8 heads over 6000, us in 1, 2, 3, 4, 5 splits: 59, 47, 55, 49, 55; over ragged
    // ones of up to 12000: 106, 69, 80, 72, 69; 64 x 5 over ragged ones of up to 2000: 47, 57, 59,
    // 61, 63).  The table's width stands for the lengths, which only the device knows: over short
    // ones in a wide table pieces are empty (one token over 500 x 12 heads 7.8 us, 15.2 in a table
    // of 2048 pages).
    const int64_t pages = c->table_pages;
    const int64_t each = p.few == 32 || p.units * (pages / 8) * 2 < cus ? 4 : 8;
    const int64_t fill = p.few == 32 ? cus : 16 * cus;
    p.splits = (int)std::min<int64_t>({std::max<int64_t>(1, fill / p.units),
                                       std::max<int64_t>(1, pages / each), kMaxSplits});
    return p;
  }
  const int64_t pack = keep ? 1 : group;
  p.tiles = tiles(pack, 128);
  p.units = p.whole = p.tiles * (keep ? q_heads : c->heads);
  // The units past a multiple of the slots (a CU is nearly as fast with one
  // workgroup as with two, so it is whole units per CU that must come out even) are cut
  // into the number of pieces that is done first, by prices from measured calls: 1.9 us
  // a page; a workgroup's start like 3 pages; for pieces 5 us of joining launch, and 0.03
  // us of the GPU's time for each piece of 128 rows written and read again.  (Of bf16 and 128
  // dims, with a full table.)  Few rows leave the page loop waiting for memory: two workgroups
  // then share a CU at full speed, and every unit may be cut.  (us with cut units / without: 8448
  // rows over 25344 x 12 heads 1170 / 1403, 40 over 20000 30.7 / 320; 5 ragged prompts, whose tiles
  // are of any lengths, 488 / 476.)
  const int64_t rows_of = std::min<int64_t>(128, (T * pack + B - 1) / B);
  const int64_t slots = rows_of <= 64 ? 2 * cus : cus, pages = c->table_pages;
  const int64_t rest = rows_of <= 64 ? p.units : p.units % cus;
  // (join_tile takes up to 128 workgroups for each unit that is cut.)
  const int64_t most = rest * 128 > kMaxBlocks
                           ? 1
                           : std::min<int64_t>(kMaxSplits, std::max<int64_t>(1, pages / 2));
  double best = 0;
  for (int64_t n = 1; n <= most; ++n) {
    const double us = (double)((rest * n + slots - 1) / slots) * (pages / (double)n + 3) * 1.9 +
                      (n > 1 ? 5 + rest * n * rows_of * (0.03 / 128) : 0);
    if (n > 1 && us >= best) continue;
    best = us;
    p.pieces = (int)n;
  }
  if (p.pieces > 1) p.whole = p.units - rest;
  return p;
}

template <int DT, int D>
void launch(const Args& a, const Plan& p, hipStream_t st) {
  const dim3 block(kThreads);
  if (p.few) {
    const dim3 grid = a.c.cu ? dim3((unsigned)(p.units * p.splits))
                             : dim3((unsigned)p.splits, (unsigned)a.c.heads,
                                    (unsigned)a.c.sequences);
    if (p.few == 16)
      hipLaunchKernelGGL((attend_few<DT, D>), grid, block, 0, st, a);
    else
      hipLaunchKernelGGL((attend_some<DT, D>), grid, block, 0, st, a);
    if (p.splits > 1)
      hipLaunchKernelGGL((join_few<DT, D>), dim3((unsigned)((int64_t)a.T * a.q_heads)), block,
                         0, st, a);
    return;
  }
  const int64_t cut = p.units - p.whole;
  hipLaunchKernelGGL((attend_tile<DT, D>), dim3((unsigned)(p.whole + cut * p.pieces)), block, 0, st,
                     a);
  if (cut > 0)
    hipLaunchKernelGGL((join_tile<DT, D>), dim3((unsigned)(cut * a.tile_rows)), block, 0, st,
                       a);
}

}  // namespace

extern "C" int64_t fvsr_paged_attn_workspace_floats(const fvsr_kv_cache* cache, int64_t T,
                                                    int64_t q_heads, int has_keep) {
  if (kv_cache_ok(cache, T) != FVSR_OK || T == 0 || cache->sequences == 0 || q_heads <= 0 ||
      q_heads > kMaxBlocks || q_heads % cache->heads)
    return 0;
  return plan_attn(cache, T, q_heads, has_keep != 0).floats(T, q_heads, cache->head_dim);
}

extern "C" int fvsr_paged_attn(const fvsr_kv_cache* cache, const void* q, int64_t q_tok_stride,
                               int64_t q_head_stride, int64_t q_heads, void* out,
                               int64_t o_tok_stride, int64_t o_head_stride, int dtype, int64_t T,
                               int causal, const uint8_t* keep, int64_t keep_q, int64_t keep_k,
                               float sm_scale, int fill_tail, float* workspace,
                               int64_t workspace_floats, void* stream) {
  const int rc = kv_cache_ok(cache, T);
  if (rc != FVSR_OK) return rc;
  if (dtype != FVSR_DT_BF16 && dtype != FVSR_DT_F16) return FVSR_EINVAL;
  if (q_heads <= 0 || q_heads % cache->heads || !(sm_scale > 0.0f) || sm_scale > 3e38f)
    return FVSR_EINVAL;
  if (keep && (keep_q < 0 || keep_k < 0)) return FVSR_EINVAL;
  if (q_heads > kMaxBlocks) return FVSR_EUNSUPPORTED;
  if (T == 0 || cache->sequences == 0) return FVSR_OK;
  if (!q || !out) return FVSR_EINVAL;
  if ((((uintptr_t)q) | (uint64_t)(q_tok_stride * 2) | (uint64_t)(q_head_stride * 2)) & 15)
    return FVSR_EUNSUPPORTED;
  if ((((uintptr_t)out) | (uint64_t)(o_tok_stride * 2) | (uint64_t)(o_head_stride * 2)) & 7)
    return FVSR_EUNSUPPORTED;
  if (T * q_heads > 0x7fffffff - 256) return FVSR_EUNSUPPORTED;
  const Plan p = plan_attn(cache, T, q_heads, keep != nullptr);
  if (p.units > kMaxBlocks / 2 || T * q_heads > kMaxBlocks * 64 ||
      (p.few && (p.units * p.splits > kMaxBlocks || (p.splits > 1 && T * q_heads > kMaxBlocks))))
    return FVSR_EUNSUPPORTED;
  const int64_t need = p.floats(T, q_heads, cache->head_dim);
  if (need && (!workspace || workspace_floats < need)) return FVSR_EWORKSPACE;
  if (need && ((uintptr_t)workspace & 15)) return FVSR_EUNSUPPORTED;
  Args a{};
  a.c = *cache;
  a.q = (const uint16_t*)q, a.out = (uint16_t*)out;
  a.q_ts = q_tok_stride, a.q_hs = q_head_stride, a.o_ts = o_tok_stride, a.o_hs = o_head_stride;
  a.keep = keep, a.keep_q = keep_q, a.keep_k = keep_k;
  a.part = workspace;
  a.scale_log2 = sm_scale * 1.4426950408889634f;
  a.T = (int)T, a.q_heads = (int)q_heads, a.group = (int)(q_heads / cache->heads);
  a.causal = causal != 0, a.splits = p.splits, a.tiles = (int)p.tiles, a.tail = fill_tail != 0;
  a.whole = (int)p.whole, a.pieces = p.pieces;
  a.tile_rows = (int)std::min<int64_t>(
      128, (cache->cu ? T : T / cache->sequences) * (keep ? 1 : a.group));
  const hipStream_t st = (hipStream_t)stream;
  const bool half = dtype == FVSR_DT_F16;
  if (cache->head_dim == 128)
    half ? launch<FVSR_DT_F16, 128>(a, p, st) : launch<FVSR_DT_BF16, 128>(a, p, st);
  else
    half ? launch<FVSR_DT_F16, 64>(a, p, st) : launch<FVSR_DT_BF16, 64>(a, p, st);
  return fvsr_launch_status();
}
