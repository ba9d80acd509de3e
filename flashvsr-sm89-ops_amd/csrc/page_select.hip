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
#include <type_traits>

#include "kv_pages.h"

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
constexpr int kNan = INT32_MIN;

// ---------------------------------------------------------------------------
// pool_kernel: a workgroup per page and head that fills up in this call.  A lane sums 16 channels
// over some of the tokens; lanes then waves join.  132 pages x 12 heads of 128 (26 MB): 7.0 us
// (3.7 TB/s; 5.0 at a copy's rate), a chain of lengths, page id, codes, the join and some 250 vector
// instructions a wave.  Without a number of rows (T -1) tables may be far wider than the lengths: a
// sequence's workgroups, some kSpread of all at most, take its pages in turn.  (64 x 4096 columns of
// 8 heads, 64 pages full in each: 86 us, 6.2 TB/s, and 4 full in each of 16 rows 19; by a workgroup to
// each column 899 and 220, and 64 x 32768 are more than a launch holds.  64 x 1000 all full, of 64
// dims, 742 and 655.  Half of kSpread: 91, 11 and 782; twice 85, 33 and 729.)
// ---------------------------------------------------------------------------
constexpr int64_t kSpread = 32 << 10;
constexpr int kMaxColumns = 32 << 10;   // of a table: one row's keys, 128 KB of LDS

struct PoolArgs {
  fvsr_kv_cache c;
  uint8_t *mean, *scale;
  int T;     // rows of the call; -1: every full page of the table
  int each;  // units of a sequence where that is the same for all (no cu, or T -1)
};

// I * 2^-e, rounded to the nearest, ties to even.
FVSR_DEV int shift_rne(int i, int e) {
  if (e <= 0) return i << min(-e, 31);
  return (i + (1 << (e - 1)) - 1 + ((i >> e) & 1)) >> e;
}

// Lanes that are equal mod L share the 2 N sums each holds: at each step a lane gives half of its
// own to the one STEP away and takes that one's part of the others.  The first of them left.
// (Steps of constant counts: a loop over both keeps the sums out of reach of constant indexes.)
template <int N, int STEP, int L>
FVSR_DEV int share(float (&s)[16], int lane) {
  if constexpr (STEP < L) {
    return 0;
  } else {
    const bool up = (lane & STEP) != 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float theirs = __shfl_xor(up ? s[i] : s[N + i], STEP);
      s[i] = (up ? s[N + i] : s[i]) + theirs;
    }
    return (up ? N : 0) + share<N / 2, STEP / 2, L>(s, lane);
  }
}

// The mean of one page and head, ph of the pool; every wave calls it.
template <int D>
FVSR_DEV void pool_page(const PoolArgs& a, int64_t ph, int (&sums)[kThreads / 64][D]) {
  constexpr int L = D / 16;            // lanes of a token's row
  constexpr int TOK = kThreads / L;    // tokens of a pass
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
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
  const int first = (lane % L) * 16 + share<8, 32, L>(s, lane);
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

template <int D>
__global__ __launch_bounds__(kThreads) void pool_kernel(PoolArgs a) {
  // (Of two pages in turn: one's are read while the next one's are made.)
  __shared__ int sums[2][kThreads / 64][D];
  const int H = (int)a.c.heads, P = (int)a.c.table_pages, B = (int)a.c.sequences;
  const int h = blockIdx.x % H, unit = blockIdx.x / H;
  const int step = a.T < 0 ? a.each : 1;
  int b, col, end;  // columns col, col + step, .. below end
  if (a.T >= 0 && a.c.cu) {
    SeqPart s;
    const auto filled = [P](int n, int len) {
      return max(0, min(len / kPage, P) - max(len - n, 0) / kPage);
    };
    if (!find_part(a.c.cu, a.c.lengths, B, a.T, unit, false, filled, s)) return;
    b = s.b, col = max(s.len - s.rows.n, 0) / kPage + s.part, end = col + 1;
  } else {
    b = unit / a.each;
    const int len = max(a.c.lengths[b], 0);
    col = unit % a.each + (a.T < 0 ? 0 : max(len - a.T / B, 0) / kPage);
    end = min(len / kPage, P);
    if (a.T >= 0) end = min(end, col + 1);
  }
  for (int buf = 0; col < end; col += step) {
    const int64_t id = a.c.table[b * a.c.table_stride + col];
    if (id >= 0 && id < a.c.pages) pool_page<D>(a, id * H + h, sums[buf]), buf ^= 1;
    if (end - col <= step) return;
  }
}

// ---------------------------------------------------------------------------
// select_kernel: a workgroup takes up to `tt` rows of a sequence and a head.  First its waves share
// out the pages, 16 at a time: products of 16 rows (a row's group padded to a power of two) and
// 16 pages; a row's largest goes to LDS as a key.  Then its waves share out the rows, and a bisection
// over the keys finds the one that just makes the list.
//
// Bound by instructions and the chain of one workgroup, not bytes: 4096 rows x 32 / 8 heads over
// some 500 pages take 40 us, 36 MB would take 7 and the products 8 (at 2058 TOP/s, what an 8192^3
// 8-bit product reaches).  Of those 30 go to q's integers and the scores (13
// instructions a row's group and page), 10 to the choice.  One row's is a chain of lengths, ids,
// means and choice: 6 us over 157 pages, 11 over 938, 16.5 over 1953; 64 rows over up to 1016
// pages each 16.7.  A tile's rows are as many as have keys in LDS at the table's width, whatever they see: the
// 4096 rows take 69 us in a table of 1024 columns, 144 in one of 4096, 856 in one of 32768.
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

// dot * 2^scale as an integer that orders like it: sign and magnitude of a float of 9 exponent
// and 20 fraction bits (|dot| < 2^21 has no more).  scale20: the scale's byte << 20.
FVSR_DEV int key_of(int dot, int scale20) {
  const uint32_t bits = __float_as_uint((float)dot);
  const int sign = dot >> 31;
  return dot == 0 ? 0 : (((int)(bits << 1 >> 4) + scale20) ^ sign) - sign;
}

// A wave's largest value, in a scalar register (DPP moves: no LDS round trips).
FVSR_DEV int wave_largest(int v) {
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0xB1, 0xf, 0xf, false));   // quad_perm [1,0,3,2]
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x4E, 0xf, 0xf, false));   // quad_perm [2,3,0,1]
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x141, 0xf, 0xf, false));  // row_half_mirror
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x140, 0xf, 0xf, false));  // row_mirror
  return max(max(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
             max(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}

// A value that just `need` of some keys reach (exact), or the largest that more do, which some
// share; at least `need` of them reach lo.  Bit by bit, in as few scalar instructions as can be.
template <class Count>
FVSR_DEV int reached(Count count, int need, int lo, int top, bool& exact) {
  for (int bit = 1 << (31 - __builtin_clz(max(top - lo, 1))); bit > 0; bit >>= 1) {
    const int n = count(lo + bit);
    lo = n >= need ? lo + bit : lo;
    if (n == need) {
      exact = true;
      return lo;
    }
  }
  exact = false;
  return lo;
}

FVSR_DEV int before(uint64_t set, int from) {  // lanes of `set` below this one, and `from`
  return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(set >> 32),
                                        __builtin_amdgcn_mbcnt_lo((uint32_t)set, from));
}

// A few powers of two below a key (keys order like floats), kLow at least: also below kNever, the
// largest key of a wave without any.
constexpr int kNear = 3 << 20;
__host__ __device__ constexpr int near_below(int key) {
  return (key > kLow + kNear ? key : kLow + kNear) - kNear;
}
static_assert(near_below(kNever) == kLow && near_below(kLow + 1) == kLow &&
                  near_below(kLow + kNear + 1) == kLow + 1 && near_below(0) == -kNear,
              "in the range of an int for every key");

// A bound that `need` of a wave's keys reach, and not many more: what `need` of the largest keys of
// 64 lanes (few are needed) or of 256 groups of them reach.  (Keys order like floats: it is
// seldom further down than near_below.)  Lanes are fewer counts (13 of 500 pages for 4096 rows: 42.2
// us, by groups 42.5; of 300 for one 7.7 and 8.0) and find no bound for many (61 of 1953: 16.6 us by
// groups, 43.3).
FVSR_DEV int bound_of(const int (&group)[4], int need) {
  const int mine = max(max(group[0], group[1]), max(group[2], group[3]));
  const int top = wave_largest(mine), near = near_below(top);
  const auto find = [&](auto reach) {
    bool exact;
    const bool fits = reach(near) >= need;
    if (!fits && reach(kLow) < need) return kLow;
    return reached(reach, need, fits ? near : kLow, top, exact);
  };
  if (need <= 16) return find([&](int at) { return (int)__popcll(__ballot(mine >= at)); });
  return find([&](int at) {
    return (int)(__popcll(__ballot(group[0] >= at)) + __popcll(__ballot(group[1] >= at)) +
                 __popcll(__ballot(group[2] >= at)) + __popcll(__ballot(group[3] >= at)));
  });
}

// A wave takes the `need` largest of n > need keys in LDS, of equal ones the first, and gives
// their places, rising, to emit(place, rank).  R: keys of a lane in registers; the others are read
// each time.  (Up to R * 64 keys are read whatever n is, in LDS and without a use.)  Those that
// reach the first bound are few as a rule: they then go to `few`, one or two to a lane (4096 rows,
// 13 of 500 pages: 40.2 us, without that 44.8; 2048 rows, 61 of 940: 52.9 and 72.6).
template <int R, class Emit>
FVSR_DEV void choose(const int* keys, int n, int need, v2i* few, Emit emit) {
  const int lane = threadIdx.x & 63;
  keys += lane;
  const auto key_at = [&](int i) { return i + lane < n ? keys[i] : kNever; };
  int key[R], group[4] = {kNever, kNever, kNever, kNever};
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int k = keys[i * 64];
    key[i] = i * 64 + lane < n ? k : kNever;
  }
#pragma unroll
  for (int i = 0; i < R; ++i) group[i % 4] = max(group[i % 4], key[i]);
  for (int i = R * 64; i < n; i += 64) group[0] = max(group[0], key_at(i));
  const auto count = [&](int at) {
    int c = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) c += __popcll(__ballot(key[i] >= at));
    for (int i = R * 64; i < n; i += 64) c += __popcll(__ballot(key_at(i) >= at));
    return c;
  };
  // Chosen: keys above lo, and the first `left` of those at it.
  int lo = bound_of(group, need), left = 0, reach = count(lo);
  if (R > 2 && reach <= 128) {
    int at = 0;
    const auto keep = [&](int i, int k) {
      const uint64_t set = __ballot(k >= lo);
      if (k >= lo) few[before(set, at)] = v2i{k, i + lane};
      at += __popcll(set);
    };
#pragma unroll
    for (int i = 0; i < R; ++i) keep(i * 64, key[i]);
    for (int i = R * 64; i < n; i += 64) keep(i, key_at(i));
    __builtin_amdgcn_wave_barrier();  // (a wave's accesses of LDS are in order)
    const auto choose_few = [&](auto lanes) {
      constexpr int F = lanes;  // of them to a lane
      int k[F], place[F], most = kNever;
#pragma unroll
      for (int f = 0; f < F; ++f) {
        const v2i x = few[f * 64 + lane];
        k[f] = f * 64 + lane < reach ? x.x : kNever, place[f] = x.y;
        most = max(most, k[f]);
      }
      const auto of_few = [&](int at) {
        int c = 0;
#pragma unroll
        for (int f = 0; f < F; ++f) c += __popcll(__ballot(k[f] >= at));
        return c;
      };
      // (By bisection while there are some to drop, then the least one by one: 4096 rows 42.2 us, by
      // bisection alone 43.5; 61 of 954 pages for 2048 rows 51.2, up to 16 one by one 55.5.)
      if (reach > need + 4) {
        bool exact;
        lo = reached(of_few, need, lo, wave_largest(most), exact);
        reach = exact ? need : of_few(lo);
      }
      while (reach > need) {
        int least = INT32_MAX;
#pragma unroll
        for (int f = 0; f < F; ++f) least = min(least, k[f] >= lo ? k[f] : INT32_MAX);
        least = ~wave_largest(~least);
        const int above = of_few(least + 1);
        lo = least, left = need - above;
        if (left > 0) break;
        lo = least + 1, left = 0, reach = above;
      }
      int at = 0;
#pragma unroll
      for (int f = 0; f < F; ++f) {
        bool in = k[f] >= lo;
        if (left > 0) {  // the first of those at lo
          const uint64_t eq = __ballot(k[f] == lo);
          in = k[f] > lo || (k[f] == lo && before(eq, 0) < left);
          left = max(left - (int)__popcll(eq), 0);
          lo += left == 0;
        }
        const uint64_t all = __ballot(in);
        if (in) emit(place[f], before(all, at));
        at += __popcll(all);
      }
    };
    if (reach <= 64)
      choose_few(std::integral_constant<int, 1>{});
    else
      choose_few(std::integral_constant<int, 2>{});
    __builtin_amdgcn_wave_barrier();
    return;
  }
  if (reach > need + 4) {
    bool exact;
    const int mine = max(max(group[0], group[1]), max(group[2], group[3]));
    lo = reached(count, need, lo, wave_largest(mine), exact);
    reach = exact ? need : count(lo);
  }
  // A few too many reach it: past the least of them, until it is those, or a tie.
  while (reach > need) {
    int least = INT32_MAX;
#pragma unroll
    for (int i = 0; i < R; ++i) least = min(least, key[i] >= lo ? key[i] : INT32_MAX);
    for (int i = R * 64; i < n; i += 64) {
      const int k = key_at(i);
      least = min(least, k >= lo ? k : INT32_MAX);
    }
    least = ~wave_largest(~least);
    const int above = count(least + 1);
    if (above < need) {
      lo = least, left = need - above;
      break;
    }
    lo = least + 1, reach = above;
  }
  if (left == 0) --lo;
  int at = 0;
  const auto put = [&](int i, int k) {
    bool in = k > lo;
    if (left > 0) {
      const uint64_t eq = __ballot(k == lo);
      in |= (k == lo) & (before(eq, 0) < left);
      left -= min(left, __popcll(eq));
    }
    const uint64_t all = __ballot(in);
    if (all == 0) return;
    if (in) emit(i + lane, before(all, at));
    at += __popcll(all);
  };
#pragma unroll
  for (int i = 0; i < R; ++i) put(i * 64, key[i]);
  for (int i = R * 64; i < n; i += 64) put(i, key_at(i));
}

// A row that has its workgroup to itself: every wave keeps those of its share of the keys that
// reach the best bound that any of them found, and one wave chooses among what is left.
constexpr int kLeft = 256;
struct Sieve {
  int bound[4], count[4];
  int key[kLeft], place[kLeft];
};
template <class Emit>
FVSR_DEV void choose_alone(const int* keys, int n, int need, int wave, Sieve& s, v2i* few,
                           Emit emit) {
  if (n <= kLeft) {
    if (wave == 0) choose<kLeft / 64>(keys, n, need, few, emit);
    return;
  }
  const int lane = threadIdx.x & 63, share = (n + 255) / 256 * 64;
  const int i0 = wave * share + lane, i1 = min(n, (wave + 1) * share);
  int group[4] = {kNever, kNever, kNever, kNever};
  for (int i = i0; i < i1; i += 256)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      group[g] = max(group[g], i + g * 64 < i1 ? keys[i + g * 64] : kNever);
  const int bound = bound_of(group, need);
  if (lane == 0) s.bound[wave] = bound;
  __syncthreads();
  const int lo = __builtin_amdgcn_readfirstlane(
      max(max(s.bound[0], s.bound[1]), max(s.bound[2], s.bound[3])));
  int c = 0;
  for (int i = i0; i < i1 + lane; i += 64)  // (whole waves)
    c += __popcll(__ballot(i < i1 && keys[min(i, n - 1)] >= lo));
  if (lane == 0) s.count[wave] = c;
  __syncthreads();
  int at = 0, total = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w == wave) at = total;
    total += s.count[w];
  }
  at = __builtin_amdgcn_readfirstlane(at), total = __builtin_amdgcn_readfirstlane(total);
  if (total > kLeft) {  // (more than a wave's lanes are wanted, or many tie)
    if (wave == 0) choose<8>(keys, n, need, few, emit);
    return;
  }
  for (int i = i0; i < i1 + lane; i += 64) {
    const int k = i < i1 ? keys[i] : kNever;
    const uint64_t in = __ballot(k >= lo);
    if (k >= lo) {
      const int to = before(in, at);
      s.key[to] = k, s.place[to] = i;
    }
    at += __popcll(in);
  }
  __syncthreads();
  if (wave != 0) return;
  if (total == need) {
    for (int i = lane; i < need; i += 64) emit(s.place[i], i);
    return;
  }
  choose<kLeft / 64>(s.key, total, need, few, [&](int i, int rank) { emit(s.place[i], rank); });
}

// A row's 16 channels at 64 w + 16 g, w < W, of one query.
template <int W>
struct Channels {
  u32x4_t raw[W][2];
  FVSR_DEV void load(Channels& c, const uint16_t* q) {
#pragma unroll
    for (int w = 0; w < W; ++w)
      c.raw[w][0] = *(const u32x4_t*)(q + 64 * w), c.raw[w][1] = *(const u32x4_t*)(q + 64 * w + 8);
  }
  // The largest magnitude's bits (of two values at once: magnitudes order like their bits).
  FVSR_DEV uint32_t largest(const Channels& c) {
    u16x2_t top = {0, 0};
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t x = c.raw[w][i >> 2][i & 3] & 0x7fff7fffu;
        top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2_t, x));
      }
    return max(top[0], top[1]);
  }
};
template <bool F16>
FVSR_DEV float half_to_f(uint32_t h) {
  if (F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)h);
  return __uint_as_float(h << 16);
}

template <int D, int GP, int M>
__global__ __launch_bounds__(kThreads) void select_kernel(SelectArgs a) {
  constexpr int W = D / 64;
  constexpr int TP = 16 / GP;  // rows of an operand
  // Groups of 16 pages at a time.  (8 in tables of more than 256 columns: 256 single tokens over up to
  // 60000 26.4 us, with 4 22.8; one over 300 pages 7.5 and 7.8, over 600 and 1953 the same.)
  constexpr int Q = 4;
  extern __shared__ __attribute__((aligned(16))) int keys[];
  __shared__ Sieve sieve;
  __shared__ v2i few[kThreads / 64][128];
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
  if (most > a.top && need > 0) {
    const int32_t* const table = a.c.table + (int64_t)s.b * a.c.table_stride;
    const int chunks = (a.group + 15) / 16;  // (more than one: GP is 16, a row to a tile)
    const uint16_t* const q0 = a.q + (int64_t)(s.rows.lo + t0) * a.q_ts + 16 * g;
    // Operand m (of rows, or of chunk c + m of one row's group) as integers.
    const auto load = [&](int m, int c, Channels<W>& x) {
      const int i = chunks == 1 ? min(m * TP + col / GP, nt - 1) : 0;
      const int head = min(chunks == 1 ? col % GP : (c + m) * 16 + col, a.group - 1);
      Channels<W>::load(x, q0 + i * a.q_ts + (int64_t)(h * a.group + head) * a.q_hs);
    };
    uint32_t top_all = 0;
    if (chunks > 1)
      for (int c = 0; c < chunks; ++c) {
        Channels<W> x;
        load(0, c, x);
        top_all = max(top_all, Channels<W>::largest(x));
      }
    const auto operand_of = [&](auto f16, int m, int c, v4i(&to)[W]) {
      constexpr bool F16 = f16;
      Channels<W> x;
      load(m, c, x);
      uint32_t top = max(top_all, Channels<W>::largest(x));
      // Over a row's lanes, then over the rows of its group.
      top = max(top, (uint32_t)__shfl_xor((int)top, 16));
      top = max(top, (uint32_t)__shfl_xor((int)top, 32));
#pragma unroll
      for (int d = 1; d < GP; d *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, d));
      // Exponent with the largest <= 127 * 2^e; 0 for all where it is not finite.
      const uint32_t t = __float_as_uint(half_to_f<F16>(top));
      const int n = t >= 0x00800000u ? (int)(t >> 23) - 127  // floor of its logarithm
                    : t != 0         ? -118 - __builtin_clz(t)
                                     : 0;
      const int e = __builtin_ldexpf(__uint_as_float(t), -n) > 127.0f / 64 ? n - 5 : n - 6;
      const bool fine = t < 0x7f800000u;
      // x * 2^-e + 1.5 * 2^23 has the nearest integer (ties to even) in its low bits: a
      // product by a power of two, in two steps where one would not hold it, and one rounding.
      const float f = __builtin_ldexpf(1.0f, min(-e, 100));
      const float f2 = __builtin_ldexpf(1.0f, -e - min(-e, 100));
#pragma unroll
      for (int w = 0; w < W; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t r[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t u = x.raw[w][i >> 1][(i & 1) * 2 + (k >> 1)];
            const float v = half_to_f<F16>(k & 1 ? u >> 16 : u & 0xffff);
            r[k] = __float_as_uint(__builtin_fmaf(F16 ? v : v * f2, f, 0x1.8p23f));
          }
          const uint32_t lo = __builtin_amdgcn_perm(r[1], r[0], 0x0c0c0400u);
          const uint32_t hi = __builtin_amdgcn_perm(r[3], r[2], 0x04000c0cu);
          to[w][i] = fine ? (int)(lo | hi) : 0;
        }
    };
    const auto operand = [&](int m, int c, v4i(&to)[W]) {
      if (a.f16)
        operand_of(std::true_type{}, m, c, to);
      else
        operand_of(std::false_type{}, m, c, to);
    };
    if (a.c.pages == 0)  // (a pool without pages)
      for (int i = threadIdx.x; i < nt * a.width; i += kThreads) keys[i] = kLow;
    for (int c = 0; c < chunks && a.c.pages > 0; c += M) {
      v4i qa[M][W];
      if constexpr (M == 1) {
        operand(0, c, qa[0]);
      } else {
        // Each wave makes one operand; they change hands where the keys will be (or, with
        // chunks, behind those).
        static_assert(M == kThreads / 64, "an operand to each wave");
        v4i* const shared_q = (v4i*)(keys + (chunks > 1 ? (a.width + 3) / 4 * 4 : 0));
        v4i own[W];
        operand(wave, c, own);
#pragma unroll
        for (int w = 0; w < W; ++w) shared_q[(wave * W + w) * 64 + lane] = own[w];
        __syncthreads();
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
          for (int w = 0; w < W; ++w) qa[m][w] = shared_q[(m * W + w) * 64 + lane];
        __syncthreads();
      }
      // 16 Q pages at a time, whose means are on their way together; the next ones' ids too.
      const auto ids = [&](int p0, int(&id)[Q]) {
#pragma unroll
        for (int k = 0; k < Q; ++k) {
          const int p = p0 + 16 * k + col;
          const int x = table[min(p, most - 1)];
          id[k] = p < most ? x : -1;
        }
      };
      int id[Q];
      ids(wave * 16 * Q, id);
      for (int p0 = wave * 16 * Q; p0 < most; p0 += kThreads / 64 * 16 * Q) {
        v4i mb[Q][W];
        int scale[Q];
#pragma unroll
        for (int k = 0; k < Q; ++k) {
          const bool there = id[k] >= 0 && id[k] < a.c.pages;
          const int64_t ph = (int64_t)(there ? id[k] : 0) * H + h;  // (no branch)
#pragma unroll
          for (int w = 0; w < W; ++w) mb[k][w] = *(const v4i*)(a.mean + ph * D + 64 * w + 16 * g);
          scale[k] = a.scale[ph] | (there ? 0 : 255);
        }
        ids(p0 + kThreads / 64 * 16 * Q, id);
        // (Bounds only where a tile has fewer rows or the last pages are at hand.)
        const bool whole = nt >= M * TP && p0 + 16 * Q <= most;
        const auto score = [&](auto checked) {
#pragma unroll
          for (int k = 0; k < Q; ++k) {
            const int p = p0 + 16 * k + col, scale20 = scale[k] << 20;
#pragma unroll
            for (int m = 0; m < M; ++m) {
              v4i x = {};
#pragma unroll
              for (int w = 0; w < W; ++w)
                x = __builtin_amdgcn_mfma_i32_16x16x64_i8(qa[m][w], mb[k][w], x, 0, 0, 0);
              // The largest over each row's group; x[j] is row 4 g + j of the operand.
              constexpr int N = GP == 1 ? 4 : GP == 2 ? 2 : 1;  // rows of the tile a lane has
              if constexpr (GP >= 2) x[0] = max(x[0], x[1]), x[2] = max(x[2], x[3]);
              if constexpr (GP == 2) x[1] = x[2];
              if constexpr (GP >= 4) x[0] = max(x[0], x[2]);
              if constexpr (GP >= 8) x[0] = max(x[0], __shfl_xor(x[0], 16));
              if constexpr (GP >= 16) x[0] = max(x[0], __shfl_xor(x[0], 32));
              const int i0 = chunks > 1 ? 0 : m * TP + (GP == 1 ? 4 * g : GP == 2 ? 2 * g
                                                        : GP == 4 ? g : GP == 8 ? g / 2 : 0);
              // (Lanes that have the same row write the same.)
#pragma unroll
              for (int n = 0; n < N; ++n) {
                int key = scale[k] == 255 ? kLow : key_of(x[n], scale20);
                int* to = &keys[(i0 + n) * a.width + p];
                if (checked && (i0 + n >= nt || p >= most)) continue;
                // (One lane has all of a page's chunks, in turn.)
                if (chunks > 1 && (c + m > 0)) key = max(key, *to);
                *to = key;
              }
            }
          }
        };
        if (chunks == 1 && whole)
          score(std::false_type{});
        else
          score(std::true_type{});
      }
    }
    __syncthreads();
  }
  const auto list = [&](int i, int first, int step, auto choice) {
    const int v = seen(i);
    int32_t* out = a.out + ((int64_t)(s.rows.lo + t0 + i) * H + h) * a.top;
    if (v <= a.top) {
      for (int c = first; c < a.top; c += step) out[c] = c < v ? c : -1;
      return;
    }
    for (int c = first; c < a.first; c += step) out[c] = c;
    for (int c = first; c < a.recent; c += step) out[a.top - a.recent + c] = v - a.recent + c;
    if (need > 0)
      choice(keys + i * a.width + a.first, v - a.first - a.recent,
             [&](int place, int rank) { out[a.first + rank] = a.first + place; });
  };
  if (M == 1 && nt == 1) {
    list(0, threadIdx.x, kThreads, [&](const int* k, int n, auto emit) {
      choose_alone(k, n, need, wave, sieve, few[wave], emit);
    });
    return;
  }
  for (int i = wave; i < nt; i += kThreads / 64)
    list(i, lane, 64, [&](const int* k, int n, auto emit) {
      if (M > 1 && most <= 128)
        choose<2>(k, n, need, few[wave], emit);
      else if (M == 1 || most <= 512)
        choose<8>(k, n, need, few[wave], emit);
      else
        choose<16>(k, n, need, few[wave], emit);
    });
}

constexpr int kLds = 64 << 10;          // of keys, at which two workgroups share a CU

template <int D, int GP>
void launch_select(const SelectArgs& a, int grid, bool many, int lds, hipStream_t st) {
  const auto run = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(kThreads), lds, st, a);
  };
  if (many)
    run(select_kernel<D, GP, 4>);
  else
    run(select_kernel<D, GP, 1>);
}

template <int D>
void launch_select(const SelectArgs& a, int gp, int grid, bool many, int lds,
                   hipStream_t st) {
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
  const int rc = kv_cache_ok(cache, T < 0 ? 0 : T, false);  // (v is not read: k is checked below)
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
  // (Any table that fvsr_select_pages takes.)
  if (T < 0 && P > kMaxColumns && B * P > kMaxBlocks) return FVSR_EUNSUPPORTED;
  // Pages that n rows can fill: one more than whole pages of them; packed, over any counts.
  const int64_t turns = std::max<int64_t>(1, kSpread / B / cache->heads);
  a.each = (int)std::min(P, T < 0 ? turns : (T / B + kPage - 1) / kPage);
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
  a.top = (int)top, a.first = (int)first, a.recent = (int)recent;
  a.f16 = dtype == FVSR_DT_F16;
  // (Widths that are odd keep rows' keys off one another's banks.)
  a.width = (int)cache->table_pages | 1;
  int gp = 1;
  while (gp < a.group && gp < 16) gp *= 2;
  // Rows of a sequence at most.
  const int64_t B = cache->sequences, each = cache->cu ? (T > B ? T : 1) : T / B;
  const int64_t fit = std::max<int64_t>(1, kLds / (a.width * 4)), tp = 16 / gp;
  // Four operands of rows share a page's means where there are rows for them and room
  // for their keys.
  const bool chunked = a.group > 16, many = chunked || (each > tp && fit > tp);
  a.tt = (int)std::min({chunked ? 1 : many ? 4 * tp : tp, fit, each});
  const int64_t tiles = cache->cu ? T / a.tt + B + 1 : B * ((each + a.tt - 1) / a.tt);
  if (tiles * cache->heads > kMaxBlocks) return FVSR_EUNSUPPORTED;
  a.tiles = (int)tiles;
  const int grid = (int)(tiles * cache->heads);
  // (Up to 512 keys are read behind a row's, 1024 behind a row that is alone.  Operands change hands
  // behind a chunked row's keys, or in place of them.)
  const int operands = many ? 4 * (int)cache->head_dim / 64 * 1024 : 0;
  const int lds = std::max({(a.tt * a.width + (a.width > 512 ? 1024 : 512)) * 4, (a.width + 1024) * 4,
                            chunked ? (a.width + 3) / 4 * 16 + operands : operands});
  const hipStream_t st = (hipStream_t)stream;
  if (cache->head_dim == 128)
    launch_select<128>(a, gp, grid, many, lds, st);
  else
    launch_select<64>(a, gp, grid, many, lds, st);
  return fvsr_launch_status();
}
