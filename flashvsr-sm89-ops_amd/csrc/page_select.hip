// Which pages of an 8-bit paged cache (kv_pages.h) a query reads.
//
// fvsr_pool_pages gives each full page and key/value head a mean key in 8 bits:
//
//   I[d] = sum over the page's 128 codes, in units of 2^-9: whole, below 2^25
//   mean[d] = rne(I[d] * 2^-e), e the least exponent with max |I| <= 127 * 2^e
//
// and 2^(e - 16) times the page's own scale is the mean's.  fvsr_select_pages scores a page
// for a row by max over the group's queries of q' . mean, q' the queries as whole numbers of
// at most 127 times one power of two.  Products of whole numbers on the matrix cores are
// exact (|dot| < 2^21), and so is a score, a whole number times a power of two: which
// pages a row reads does not hang on the order of a sum, and equal scores are equal.  Only
// full pages need one: the page that holds a row's own position is always read.
#include <algorithm>

#include "kv_pages.h"

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
constexpr int kNan = INT32_MIN;

// ---------------------------------------------------------------------------
// pool_kernel: a workgroup per page and head that fills up in this call.
// ---------------------------------------------------------------------------
struct PoolArgs {
  fvsr_kv_cache c;
  uint8_t *mean, *scale;
  int T;     // rows of the call; -1: every full page of the table
  int each;  // units of a sequence where that is the same for all (no cu)
};

// I * 2^-e, rounded to the nearest, ties to even.
FVSR_DEV int shift_rne(int i, int e) {
  if (e <= 0) return i << min(-e, 31);
  return (i + (1 << (e - 1)) - 1 + ((i >> e) & 1)) >> e;
}

template <int D>
__global__ __launch_bounds__(kThreads) void pool_kernel(PoolArgs a) {
  constexpr int L = D / 16;            // lanes of a token's row
  constexpr int TOK = kThreads / L;    // tokens of a pass
  __shared__ int sums[kThreads / 64][D];
  const int H = (int)a.c.heads, P = (int)a.c.table_pages, B = (int)a.c.sequences;
  const int h = blockIdx.x % H, unit = blockIdx.x / H;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int b, col;
  if (a.T >= 0 && a.c.cu) {
    SeqPart s;
    const auto filled = [P](int n, int len) {
      return max(0, min(len / kPage, P) - max(len - n, 0) / kPage);
    };
    if (!find_part(a.c.cu, a.c.lengths, B, a.T, unit, false, filled, s)) return;
    b = s.b, col = max(s.len - s.rows.n, 0) / kPage + s.part;
  } else {
    b = unit / a.each;
    const int len = max(a.c.lengths[b], 0);
    col = unit % a.each + (a.T < 0 ? 0 : max(len - a.T / B, 0) / kPage);
    if (col >= min(len / kPage, P)) return;
  }
  const int64_t id = a.c.table[b * a.c.table_stride + col];
  if (id < 0 || id >= a.c.pages) return;
  const int64_t ph = id * H + h;
  const uint8_t* kp = (const uint8_t*)a.c.k + ph * kPage * D + threadIdx.x * 16;
  u32x4_t w[kPage / TOK];
#pragma unroll
  for (int t = 0; t < kPage / TOK; ++t) w[t] = *(const u32x4_t*)(kp + t * TOK * D);
  const int ks = ((const uint8_t*)a.c.k_scale)[ph];
  // 16 channels of 2 or 4 tokens a lane, then of 32: below 2^24 units, so exact in fp32.
  float s[16] = {};
#pragma unroll
  for (int t = 0; t < kPage / TOK; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const v2f lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[t][i], false);
      const v2f hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[t][i], true);
      s[4 * i] += lo[0], s[4 * i + 1] += lo[1], s[4 * i + 2] += hi[0], s[4 * i + 3] += hi[1];
    }
  // Lanes of one place in the row (equal mod L) halve the channels they hold at each step.
  int first = (lane % L) * 16;
#pragma unroll
  for (int step = 32, n = 8; step >= L; step /= 2, n /= 2) {
    const bool up = (lane & step) != 0;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float theirs = __shfl_xor(up ? s[i] : s[n + i], step);
      s[i] = (up ? s[n + i] : s[i]) + theirs;
    }
    if (up) first += n;
  }
  constexpr int R = 16 * L / 64;  // channels left to a lane
#pragma unroll
  for (int i = 0; i < R; ++i)
    sums[wave][first + i] = s[i] == s[i] ? (int)(s[i] * 512.0f) : kNan;
  __syncthreads();
  if (wave != 0) return;
  constexpr int C = D / 64;
  int total[C], top = 0;
  bool bad = ks == 255;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    total[c] = 0;
#pragma unroll
    for (int v = 0; v < kThreads / 64; ++v) {
      const int x = sums[v][lane * C + c];
      bad |= x == kNan;
      total[c] += x == kNan ? 0 : x;
    }
    top = max(top, abs(total[c]));
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) top = max(top, __shfl_xor(top, d));
  const int own = ks - 127 - 16;  // exponent of a unit of I
  int e = -127 - own;             // the least there is
  if (top > 0) {
    const int x = 31 - __builtin_clz(top);
    e = max(e, ((int64_t)top << 6) <= ((int64_t)127 << x) ? x - 6 : x - 5);
  }
  e = min(e, 127 - own);  // (scales near 2^127 alone: means past it are held there)
  const bool none = __ballot(bad) != 0;  // a NaN code or scale: no mean, and a scale that says so
  uint8_t* mp = a.mean + ph * D + lane * C;
#pragma unroll
  for (int c = 0; c < C; ++c)
    total[c] = none ? 0 : min(max(shift_rne(total[c], e), -127), 127);
  if (C == 2)
    *(uint16_t*)mp = (uint16_t)((total[0] & 255) | (total[C - 1] & 255) << 8);
  else
    *mp = (uint8_t)total[0];
  if (lane == 0) a.scale[ph] = (uint8_t)(none ? 255 : e + own + 127);
}

// ---------------------------------------------------------------------------
// select_kernel: a workgroup takes up to `tt` rows of a sequence and a head.  First its waves
// share out the pages, 16 at a time: products of 16 rows (a row's group padded to a power
// of two) and 16 pages; a row's largest goes to LDS as a key.  Then its waves share out the rows:
// a bisection over the keys finds the one that just makes the list.
//
// Operands of v_mfma_i32_16x16x64_i8: lane (r, g) = (l % 16, l / 16) holds bytes 16 g .. of row r;
// accumulator j of lane (c, g) is row 4 g + j (a query) of column c (a page).
// ---------------------------------------------------------------------------
struct SelectArgs {
  fvsr_kv_cache c;
  const int8_t* mean;
  const uint8_t* scale;
  const uint16_t* q;
  int64_t q_ts, q_hs;
  int32_t* out;
  int T, group, top, first, recent, f16;
  int tt, tiles, width;  // rows of a tile; tiles of all sequences; keys of a row in LDS
};

constexpr int kLow = -(1 << 30);  // key of a page without a mean: below any other
constexpr int kNever = INT32_MIN;

// dot * 2^scale as an integer that orders like it: sign and magnitude of a float of 9
// exponent and 20 fraction bits (|dot| < 2^21 has no more).
FVSR_DEV int key_of(int dot, int scale) {
  const uint32_t bits = __float_as_uint((float)abs(dot)) >> 3;
  const int key = (int)(bits + ((uint32_t)scale << 20));
  return dot == 0 ? 0 : dot < 0 ? -key : key;
}

FVSR_DEV float q_at(uint32_t pair, int odd, int f16) {
  const uint16_t u = (uint16_t)(odd ? pair >> 16 : pair & 0xffff);
  return f16 ? (float)__builtin_bit_cast(_Float16, u) : bf2f(u);
}

// What `n` waves that work on one row tell one another.
struct Told {
  int count[2][4], gt[4], eq[4], top[4], low[4];
};

// The list of a row that sees the columns 0 .. seen - 1, more than `top` of them.
template <int WAVES>
FVSR_DEV void pick(const SelectArgs& a, const int* keys, int seen, int wave, Told& told,
                   int32_t* out) {
  constexpr int R = 8;
  const int lane = threadIdx.x & 63;
  const int share = WAVES == 1 ? seen : (seen + 64 * WAVES - 1) / (64 * WAVES) * 64;
  const int c0 = min(seen, wave * share), c1 = min(seen, c0 + share);
  const int need = a.top - a.first - a.recent, end = seen - a.recent;
  const auto key_at = [&](int c) { return c >= a.first && c < min(end, c1) ? keys[c] : kNever; };
  int key[R], top = kNever;
#pragma unroll
  for (int i = 0; i < R; ++i) top = max(top, key[i] = key_at(c0 + i * 64 + lane));
  for (int c = c0 + R * 64; c < c1; c += 64) top = max(top, key_at(c + lane));
  // Every lane's largest is at least `low`: with 64 of them (or more) one bound of the search.
  int low = top;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    top = max(top, __shfl_xor(top, d));
    low = min(low, __shfl_xor(low, d));
  }
  if (WAVES > 1) {
    if (lane == 0) told.top[wave] = top, told.low[wave] = low;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = max(top, told.top[w]), low = min(low, told.low[w]);
  }
  top = __builtin_amdgcn_readfirstlane(top);
  low = __builtin_amdgcn_readfirstlane(low);
  int turn = 0;
  const auto count = [&](int at) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) n += __popcll(__ballot(key[i] >= at));
    for (int c = c0 + R * 64; c < c1; c += 64) n += __popcll(__ballot(key_at(c + lane) >= at));
    if (WAVES > 1) {
      if (lane == 0) told.count[turn & 1][wave] = n;
      __syncthreads();
      n = 0;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) n += told.count[turn & 1][w];
      ++turn;
    }
    return __builtin_amdgcn_readfirstlane(n);
  };
  // At least `need` keys are >= lo, fewer are >= hi; `above` of them.
  int lo = need <= 64 * WAVES && low > kLow ? low : kLow, hi = top + 1, above = 0;
  int ties = need;
  if (need > 0) {
    while (hi - lo > 1) {
      const int mid = lo + (hi - lo) / 2, n = count(mid);
      if (n == need) {  // no tie to break: all above mid - 1
        lo = mid - 1, above = need;
        break;
      }
      if (n > need)
        lo = mid;
      else
        hi = mid, above = n;
    }
    ties = need - above;
  } else {
    lo = top;  // none above
    ties = 0;
  }
  // Columns in the list: those always there, keys above lo, the first `ties` at lo.
  const auto sure = [&](int c) { return c < c1 && (c < a.first || c >= end); };
  int at = 0, left = ties;
  if (WAVES > 1) {
    int gt = 0, eq = 0;
    for (int c = c0; c < c1; c += 64) {
      const int k = key_at(c + lane);
      gt += __popcll(__ballot(sure(c + lane) || k > lo));
      eq += __popcll(__ballot(k == lo));
    }
    if (lane == 0) told.gt[wave] = gt, told.eq[wave] = eq;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w)
      if (w < wave) {
        const int took = min(left, told.eq[w]);
        at += told.gt[w] + took, left -= took;
      }
  }
  const uint64_t below = (1ull << lane) - 1;
  for (int c = c0; c < c1; c += 64) {
    const int k = key_at(c + lane);
    const bool tie = k == lo;
    const uint64_t eq = __ballot(tie);
    const bool in = sure(c + lane) || k > lo || (tie && __popcll(eq & below) < left);
    const uint64_t all = __ballot(in);
    if (in) out[at + __popcll(all & below)] = c + lane;
    at += __popcll(all);
    left -= min(left, __popcll(eq));
  }
}

template <int D, int GP, int M>
__global__ __launch_bounds__(kThreads) void select_kernel(SelectArgs a) {
  constexpr int W = D / 64;
  constexpr int TP = 16 / GP;  // rows of an operand
  extern __shared__ int keys[];
  __shared__ Told told;
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int H = (int)a.c.heads, P = (int)a.c.table_pages, B = (int)a.c.sequences;
  // Tiles of one head are neighbours on one XCD, which read the same means.
  const int total = (int)gridDim.x, wg = blockIdx.x;
  const int per = total / 8, rem = total % 8, xcd = wg % 8, loc = wg / 8;
  const int at = xcd < rem ? xcd * (per + 1) + loc : rem * (per + 1) + (xcd - rem) * per + loc;
  const int h = at / a.tiles;
  SeqPart s;
  if (a.c.cu) {
    const int tt = a.tt;
    const auto tiles_of = [tt](int n, int) { return (n + tt - 1) / tt; };
    if (!find_part(a.c.cu, a.c.lengths, B, a.T, at % a.tiles, true, tiles_of, s)) return;
  } else {
    const int each = a.tiles / B;
    s.b = at % a.tiles / each, s.part = at % a.tiles % each;
    s.rows = seq_rows(nullptr, s.b, B, a.T);
    s.len = max(a.c.lengths[s.b], 0);
  }
  const int t0 = s.part * a.tt, nt = min(a.tt, s.rows.n - t0);
  // Columns that row i of the tile sees.
  const auto seen = [&](int i) {
    const int p = s.len - s.rows.n + t0 + i;
    return p < 0 ? 0 : min(p / kPage + 1, P);
  };
  const int most = seen(nt - 1), need = a.top - a.first - a.recent;
  const int32_t* const table = a.c.table + (int64_t)s.b * a.c.table_stride;
  if (most > a.top && need > 0) {
    const int chunks = (a.group + 15) / 16;  // (more than one: GP is 16, a row to a tile)
    const uint16_t* const q0 = a.q + (int64_t)(s.rows.lo + t0) * a.q_ts;
    const auto row_of = [&](int m, int c) {
      const int i = chunks == 1 ? min(m * TP + col / GP, nt - 1) : 0;
      const int head = min(chunks == 1 ? col % GP : (c + m) * 16 + col, a.group - 1);
      return (const u32x4_t*)(q0 + i * a.q_ts + (int64_t)(h * a.group + head) * a.q_hs + 16 * g);
    };
    const auto load = [&](int m, int c, u32x4_t(&raw)[W][2]) {
      const u32x4_t* p = row_of(m, c);
#pragma unroll
      for (int w = 0; w < W; ++w) raw[w][0] = p[8 * w], raw[w][1] = p[8 * w + 1];
    };
    const auto largest = [&](const u32x4_t(&raw)[W][2]) {
      uint32_t top = 0;
#pragma unroll
      for (int w = 0; w < W; ++w)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          top = max(top, __float_as_uint(q_at(raw[w][i >> 3][(i >> 1) & 3], i & 1, a.f16)) &
                             0x7fffffffu);
      return top;
    };
    uint32_t top_all = 0;
    if (chunks > 1)
      for (int c = 0; c < chunks; ++c) {
        u32x4_t raw[W][2];
        load(0, c, raw);
        top_all = max(top_all, largest(raw));
      }
    for (int c = 0; c < chunks; c += M) {
      v4i qa[M][W];
#pragma unroll
      for (int m = 0; m < M; ++m) {
        u32x4_t raw[W][2];
        load(m, c, raw);
        uint32_t top = max(top_all, largest(raw));
        // Over a row's lanes, then over the rows of its group.
        top = max(top, (uint32_t)__shfl_xor((int)top, 16));
        top = max(top, (uint32_t)__shfl_xor((int)top, 32));
#pragma unroll
        for (int d = 1; d < GP; d *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, d));
        // Exponent with top <= 127 * 2^e; 0 for all where it is not finite.
        const float t = __uint_as_float(top);
        const int x = top >= 0x00800000u ? (int)(top >> 23) - 127  // floor of its logarithm
                      : top != 0         ? -118 - __builtin_clz(top)
                                         : 0;
        const int e = __builtin_ldexpf(t, -x) > 127.0f / 64 ? x - 5 : x - 6;
        const bool fine = top < 0x7f800000u;
#pragma unroll
        for (int w = 0; w < W; ++w)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t word = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int n = 4 * i + k;
              const float v = q_at(raw[w][n >> 3][(n >> 1) & 3], n & 1, a.f16);
              const int r = fine ? (int)__builtin_rintf(__builtin_ldexpf(v, -e)) : 0;
              word |= ((uint32_t)r & 255u) << (8 * k);
            }
            qa[m][w][i] = (int)word;
          }
      }
      for (int p0 = wave * 16; p0 < most; p0 += kThreads / 64 * 16) {
        const int p = p0 + col;
        const int id = p < most ? table[p] : -1;
        const bool there = id >= 0 && id < a.c.pages;
        const int64_t ph = (int64_t)(there ? id : 0) * H + h;
        v4i mb[W];
#pragma unroll
        for (int w = 0; w < W; ++w) mb[w] = v4i{};
        int scale = 255;
        if (there) {
#pragma unroll
          for (int w = 0; w < W; ++w) mb[w] = *(const v4i*)(a.mean + ph * D + 64 * w + 16 * g);
          scale = a.scale[ph];
        }
#pragma unroll
        for (int m = 0; m < M; ++m) {
          v4i x = {};
#pragma unroll
          for (int w = 0; w < W; ++w)
            x = __builtin_amdgcn_mfma_i32_16x16x64_i8(qa[m][w], mb[w], x, 0, 0, 0);
          // The largest over each row's group; x[j] is row 4 g + j of the operand.
          constexpr int N = GP == 1 ? 4 : GP == 2 ? 2 : 1;  // rows of the tile a lane has
          if constexpr (GP >= 2) x[0] = max(x[0], x[1]), x[2] = max(x[2], x[3]);
          if constexpr (GP == 2) x[1] = x[2];
          if constexpr (GP >= 4) x[0] = max(x[0], x[2]);
          if constexpr (GP >= 8) x[0] = max(x[0], __shfl_xor(x[0], 16));
          if constexpr (GP >= 16) x[0] = max(x[0], __shfl_xor(x[0], 32));
          const int i0 = chunks > 1 ? 0 : m * TP + (GP == 1 ? 4 * g : GP == 2 ? 2 * g
                                                    : GP == 4 ? g : GP == 8 ? g / 2 : 0);
          const bool mine = GP <= 4 || (GP == 8 ? (g & 1) == 0 : g == 0);
#pragma unroll
          for (int n = 0; n < N; ++n) {
            if (!mine || i0 + n >= nt || p >= most) continue;
            int key = scale == 255 ? kLow : key_of(x[n], scale);
            int* to = &keys[(i0 + n) * a.width + p];
            // (One lane has all of a page's chunks, in turn.)
            if (chunks > 1 && (c + m > 0)) key = max(key, *to);
            *to = key;
          }
        }
      }
    }
    __syncthreads();
  }
  const auto write = [&](int i, int first, int step, bool together) {
    const int v = seen(i);
    int32_t* out = a.out + ((int64_t)(s.rows.lo + t0 + i) * H + h) * a.top;
    if (v <= a.top)
      for (int c = first; c < a.top; c += step) out[c] = c < v ? c : -1;
    else if (together)
      pick<4>(a, keys + i * a.width, v, wave, told, out);
    else
      pick<1>(a, keys + i * a.width, v, 0, told, out);
  };
  if (nt == 1)
    write(0, threadIdx.x, kThreads, true);
  else
    for (int i = wave; i < nt; i += kThreads / 64) write(i, lane, 64, false);
}

constexpr int kLds = 64 << 10;          // of keys, at which two workgroups share a CU
constexpr int kMaxColumns = 32 << 10;   // one row's keys: 128 KB

template <int D, int GP>
void launch_select(SelectArgs& a, int grid, bool many, int lds, hipStream_t st) {
  if (many)
    hipLaunchKernelGGL((select_kernel<D, GP, 4>), dim3(grid), dim3(kThreads), lds, st, a);
  else
    hipLaunchKernelGGL((select_kernel<D, GP, 1>), dim3(grid), dim3(kThreads), lds, st, a);
}

template <int D>
void launch_select(SelectArgs& a, int gp, int grid, bool many, int lds, hipStream_t st) {
  switch (gp) {
    case 1: return launch_select<D, 1>(a, grid, many, lds, st);
    case 2: return launch_select<D, 2>(a, grid, many, lds, st);
    case 4: return launch_select<D, 4>(a, grid, many, lds, st);
    case 8: return launch_select<D, 8>(a, grid, many, lds, st);
    default: return launch_select<D, 16>(a, grid, many, lds, st);
  }
}

}  // namespace

extern "C" int fvsr_pool_pages(const fvsr_kv_cache* cache, void* mean, void* mean_scale, int64_t T,
                               void* stream) {
  const int rc = kv_cache_ok(cache, T < 0 ? 0 : T);
  if (rc != FVSR_OK) return rc;
  if (T < -1) return FVSR_EINVAL;
  const int64_t B = cache->sequences, P = cache->table_pages;
  if (B == 0 || T == 0 || P == 0 || cache->pages == 0) return FVSR_OK;
  if (!cache->k || !cache->k_scale || !cache->table || !cache->lengths || !mean || !mean_scale)
    return FVSR_EINVAL;
  if (((uintptr_t)cache->k | (uintptr_t)mean) & 15) return FVSR_EUNSUPPORTED;
  PoolArgs a{};
  a.c = *cache;
  a.mean = (uint8_t*)mean, a.scale = (uint8_t*)mean_scale;
  a.T = (int)T;
  // Pages that n rows can fill: one more than whole pages of them; packed, over any counts.
  a.each = (int)(T < 0 ? P : std::min(P, (T / B + kPage - 1) / kPage));
  const int64_t units = T >= 0 && cache->cu ? (T + B * (kPage - 1)) / kPage : B * a.each;
  if (units > kMaxBlocks || units * cache->heads > kMaxBlocks) return FVSR_EUNSUPPORTED;
  if (units == 0) return FVSR_OK;
  const dim3 grid((unsigned)(units * cache->heads));
  const hipStream_t st = (hipStream_t)stream;
  if (cache->head_dim == 128)
    hipLaunchKernelGGL(pool_kernel<128>, grid, dim3(kThreads), 0, st, a);
  else
    hipLaunchKernelGGL(pool_kernel<64>, grid, dim3(kThreads), 0, st, a);
  return fvsr_launch_status();
}

extern "C" int fvsr_select_pages(const fvsr_kv_cache* cache, const void* mean,
                                 const void* mean_scale, const void* q, int64_t q_tok_stride,
                                 int64_t q_head_stride, int64_t q_heads, int dtype, int64_t T,
                                 int64_t top, int64_t first, int64_t recent, int32_t* columns,
                                 void* stream) {
  const int rc = kv_cache_ok(cache, T, false);
  if (rc != FVSR_OK) return rc;
  if (dtype != FVSR_DT_BF16 && dtype != FVSR_DT_F16) return FVSR_EINVAL;
  if (q_heads <= 0 || q_heads % cache->heads || first < 0 || recent < 1 || top < first + recent)
    return FVSR_EINVAL;
  if (q_heads > kMaxBlocks || top > 0xffffff || cache->table_pages > kMaxColumns)
    return FVSR_EUNSUPPORTED;
  if (T == 0 || cache->sequences == 0) return FVSR_OK;
  if (!q || !columns || (cache->pages > 0 && (!mean || !mean_scale))) return FVSR_EINVAL;
  if (((uintptr_t)q | (uintptr_t)mean | (uint64_t)(q_tok_stride * 2) |
       (uint64_t)(q_head_stride * 2)) & 15)
    return FVSR_EUNSUPPORTED;
  SelectArgs a{};
  a.c = *cache;
  a.mean = (const int8_t*)mean, a.scale = (const uint8_t*)mean_scale;
  a.q = (const uint16_t*)q, a.q_ts = q_tok_stride, a.q_hs = q_head_stride;
  a.out = columns;
  a.T = (int)T, a.group = (int)(q_heads / cache->heads);
  a.top = (int)top, a.first = (int)first, a.recent = (int)recent, a.f16 = dtype == FVSR_DT_F16;
  // (Widths that are odd keep rows' keys off one another's banks.)
  a.width = (int)cache->table_pages | 1;
  int gp = 1;
  while (gp < a.group && gp < 16) gp *= 2;
  const int64_t B = cache->sequences, each = cache->cu ? T : T / B;
  const int64_t fit = std::max<int64_t>(1, kLds / (a.width * 4)), tp = 16 / gp;
  // Four operands of rows share a page's means where there are rows for them and room
  // for their keys.
  const bool chunked = a.group > 16, many = chunked || (each > tp && fit > tp);
  a.tt = (int)std::min({chunked ? 1 : many ? 4 * tp : tp, fit, each});
  const int64_t tiles = cache->cu ? T / a.tt + B + 1 : B * ((each + a.tt - 1) / a.tt);
  if (tiles * cache->heads > kMaxBlocks) return FVSR_EUNSUPPORTED;
  a.tiles = (int)tiles;
  const int grid = (int)(tiles * cache->heads), lds = a.tt * a.width * 4;
  const hipStream_t st = (hipStream_t)stream;
  if (cache->head_dim == 128)
    launch_select<128>(a, gp, grid, many, lds, st);
  else
    launch_select<64>(a, gp, grid, many, lds, st);
  return fvsr_launch_status();
}
