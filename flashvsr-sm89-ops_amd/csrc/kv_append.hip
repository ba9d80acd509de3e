// Keys and values into an 8-bit paged cache: RMSNorm and rotation of k (and
// of q, which goes back in its own type), quantisation to e4m3 with one
// power-of-two scale for a page (128 tokens) and head.
//
//   x = rotate(k * rsqrt(mean(k^2) + eps) * w)       fp32, mean over a head or the whole row
//   e = least exponent >= -126 with max |x| <= 448 * 2^e over the page's new, finite values;
//       not below the page's own where it holds tokens before them
//   code = e4m3(x * 2^-e), held codes e4m3(code * 2^(e_old - e))
//
// A power of two costs no precision (e4m3 is a floating format), makes the
// scale the matrix cores' own scale operand, and lets a growing page round its
// held codes again without loss unless they become subnormal.  The rotation pairs
// neighbours (2i, 2i + 1), as fvsr_rms_rope does, and nothing is rounded between
// the norm and the code (q: the output).
//
// One workgroup per (page, head) and k or v: a page's scale needs all of its new
// tokens at once, and 128 x 128 values fit a workgroup's registers, so they are
// read once.  Thread t holds dims 8*(t % (D/8)).. of 4 consecutive tokens; v's codes
// turn to [dim][token] through LDS.  The q rows are further workgroups of the
// same launch.  An RMSNorm over whole rows needs other heads' values: the rows'
// statistics come from a launch before (which also does v), or, for a few
// tokens, each workgroup sums its own rows.  Up to 8 tokens of each sequence go by
// waves instead, without LDS or barriers.
//
// Measured, q with k and v: one token x 12 heads 5.5 us (latency: a chain of four loads),
// 192 of 32/8 heads 6.0; 24 ragged prompts of 6119 tokens in all x 16/4 heads of 64, fp16
// 10.5 us (3.5 TB/s); 16896 tokens x 12 heads with row norms 73 us (3.7 TB/s; 5.1 is a copy's
// rate, and k's second read is not counted), in fp32 128 (3.7).  Between them a page's chain of
// loads bounds it: lengths, page id and positions, rows, rotations, codes.
#include <algorithm>
#include <type_traits>

#include "kv_pages.h"

namespace {

constexpr int kThreads = 256;  // kv_token_kernel
constexpr int kTokens = 4;     // tokens of a thread of a page's workgroup
template <int D>
constexpr int kWg = kPage / kTokens * (D / 8);  // its threads: 512 or 256
enum { kNone = FVSR_NORM_NONE, kHead = FVSR_NORM_HEAD, kRow = FVSR_NORM_ROW };

struct Args {
  fvsr_kv_cache c;
  const void *k, *v, *q, *k_weight, *q_weight;
  void* q_out;
  const float* cs;           // [cs_rows][D/2][2] (cos, sin); null: no rotation
  const int32_t* positions;  // row of cs for each token; null: the token's own number
  double* row_stat;          // 1/rms of each k row (row norm, from the launch before)
  double k_per;              // 1 / elements that a norm of k is over
  int64_t k_ts, k_hs, v_ts, v_hs, q_ts, q_hs, cs_rows;
  int T, q_heads, k_norm, q_norm, w_dt, units, units_max, page_wgs;
  float eps;
};

// Eight consecutive elements as they lie in memory (16-byte aligned).
template <int DT>
struct Raw8 {
  u32x4_t w[DT == FVSR_DT_F32 ? 2 : 1];
};
template <int DT>
FVSR_DEV Raw8<DT> load_raw(const void* p, int64_t i) {
  const u32x4_t* s = (const u32x4_t*)((const uint8_t*)p + i * (DT == FVSR_DT_F32 ? 4 : 2));
  Raw8<DT> r;
  r.w[0] = s[0];
  if constexpr (DT == FVSR_DT_F32) r.w[1] = s[1];
  return r;
}
template <int DT>
FVSR_DEV void widen(const Raw8<DT>& r, float (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if constexpr (DT == FVSR_DT_F32) {
      x[e] = __uint_as_float(r.w[e >> 2][e & 3]);
    } else {
      const uint32_t u = r.w[0][e >> 1];
      if constexpr (DT == FVSR_DT_F16)
        x[e] = (float)__builtin_bit_cast(_Float16, (uint16_t)(e & 1 ? u >> 16 : u));
      else
        x[e] = e & 1 ? bf_hi(u) : bf_lo(u);
    }
  }
}
FVSR_DEV void load8(const void* p, int dt, int64_t i, float (&x)[8]) {
  if (dt == FVSR_DT_F32)
    widen(load_raw<FVSR_DT_F32>(p, i), x);
  else if (dt == FVSR_DT_F16)
    widen(load_raw<FVSR_DT_F16>(p, i), x);
  else
    widen(load_raw<FVSR_DT_BF16>(p, i), x);
}

FVSR_DEV void store8(void* p, int dt, int64_t i, const float (&x)[8]) {
  if (dt == FVSR_DT_F32) {
    f32x4_t* s = (f32x4_t*)((float*)p + i);
    s[0] = f32x4_t{x[0], x[1], x[2], x[3]};
    s[1] = f32x4_t{x[4], x[5], x[6], x[7]};
  } else if (dt == FVSR_DT_F16) {
    typedef _Float16 h8 __attribute__((ext_vector_type(8)));
    h8 a;
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e] = (_Float16)x[e];
    *(h8*)((_Float16*)p + i) = a;
  } else {
    *(u32x4_t*)((uint16_t*)p + i) =
        u32x4_t{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                pack_bf16x2(x[6], x[7])};
  }
}

// Sums and what follows from them in fp32, or (T double) in 64 bits.  q is rounded to its
// own type in the end, where fp32's steps do not show, but k to a code of 4 bits: fp32's
// steps put 1 or 2 in 10^6 on the other side of a border between codes, 1 / 16 off.  So
// k's sums are taken in 64 bits (beyond eight squares at least, which also keeps those that
// fp32 does not hold), and what lies near a border is computed again in 64 bits.  (16896
// tokens x 12 heads: errors of k against 64 bits 2e-5 of its norm without that, 1e-7 so; 70.7 us
// without, 73.3 so.  6119 tokens in ragged prompts 10.0 us, 10.6.)
template <class T>
FVSR_DEV T sum_sq(const float (&x)[8]) {
  T s = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) s += (T)x[e] * (T)x[e];
  return s;
}

FVSR_DEV float inv_rms(float sq, int n, float eps) { return 1.0f / __builtin_sqrtf(sq / n + eps); }
// The same in 64 bits, with per = 1 / n: the instruction's 2^-23 and a Newton step, 2^-45.
FVSR_DEV double inv_rms64(double sq, double per, float eps) {
  const double m = __builtin_fma(sq, per, (double)eps), r = __builtin_amdgcn_rsq(m);
  const double e = __builtin_fma(-0.5 * m * r, r, 0.5);
  return e == e ? __builtin_fma(r, e, r) : r;  // (m 0 or infinite: r is it)
}

// Sum over the N = 8, 16 or 64 lanes around, from lane to lane (dpp).
template <int CTRL, int ROWS = 0xf>
FVSR_DEV float moved(float v) {
  return dpp_f32<CTRL, ROWS>(v);
}
template <int CTRL, int ROWS = 0xf>
FVSR_DEV double moved(double v) {
  typedef float v2f __attribute__((ext_vector_type(2)));
  const v2f u = __builtin_bit_cast(v2f, v);
  return __builtin_bit_cast(double, v2f{dpp_f32<CTRL, ROWS>(u[0]), dpp_f32<CTRL, ROWS>(u[1])});
}
FVSR_DEV double lane63(double v) {
  typedef float v2f __attribute__((ext_vector_type(2)));
  const v2f u = __builtin_bit_cast(v2f, v);
  return __builtin_bit_cast(double, v2f{::lane63(u[0]), ::lane63(u[1])});
}
template <int N, class T>
FVSR_DEV T lanes_sum(T v) {
  v += moved<0xB1>(v);   // quad_perm [1,0,3,2]
  v += moved<0x4E>(v);   // quad_perm [2,3,0,1]
  v += moved<0x141>(v);  // row_half_mirror
  if constexpr (N > 8) v += moved<0x140>(v);  // row_mirror
  if constexpr (N > 16) {
    v += moved<0x142, 0xa>(v);  // row_bcast:15 into rows 1, 3
    v += moved<0x143, 0xc>(v);  // row_bcast:31 into rows 2, 3
    v = lane63(v);
  }
  return v;
}

// Whether one of the values seen lies within kNear fp32 steps of a border between
// codes of 4 bits (subnormal codes aside, whose steps are small): mantissas whose last 20
// bits are near their half.  In units of 2^-24 of itself a value is off by half of what
// its sum of squares is (8, where eight at a time are summed in fp32) and 1 for 1 / rms as fp32,
// alike in both terms of a rotation, 3 in each term (x r, w, cos or sin) and 1 in the result:
// 5 + 3 / 0.7 + 1 < 11 steps where the rotation leaves 0.7 of its terms.
constexpr uint32_t kNear = 12;
struct Border {
  uint32_t least = ~0u;
  __device__ __forceinline__ void see(float x) {
    least = min(least, (__float_as_uint(x) << 12) + ((kNear << 12) - 0x80000000u));
  }
  __device__ __forceinline__ bool near() const { return least < 2 * kNear << 12; }
};

// d as fp32 with its last bit set if anything is cut off: the code that it rounds to is the
// one that d itself would.
FVSR_DEV float to_odd(double d) {
  const float f = (float)d;
  const double back = f;
  uint32_t u = __float_as_uint(f);
  u -= __builtin_fabs(back) > __builtin_fabs(d);
  u |= back != d && back == back;
  return __uint_as_float(u);
}

// A whole row of H heads by one wave: the first N pieces of eight per lane go out
// together and stay in registers.  Returns the sum of squares.
template <class T, int DT, int D, int N>
FVSR_DEV T load_row(const void* x, int64_t row, int64_t hs, int H, Raw8<DT> (&held)[N]) {
  constexpr int C = D / 8;
  const int lane = threadIdx.x & 63, n = H * C;
  const auto at = [&](int c) { return row + (c / C) * hs + (c % C) * 8; };
#pragma unroll
  for (int i = 0; i < N; ++i) {
    held[i] = Raw8<DT>{};
    if (lane + 64 * i < n) held[i] = load_raw<DT>(x, at(lane + 64 * i));
  }
  T s = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float a[8];
    widen(held[i], a);
    s += sum_sq<T>(a);
  }
  for (int c = lane + 64 * N; c < n; c += 64) {
    float a[8];
    load8(x, DT, at(c), a);
    s += sum_sq<T>(a);
  }
  return lanes_sum<64>(s);
}
template <int DT, int D, int N>
FVSR_DEV double row_sq(const void* x, int64_t row, int64_t hs, int H) {
  Raw8<DT> held[N];
  return load_row<double, DT, D>(x, row, hs, H, held);
}

// A position outside the table gives NaN (every result has a cosine in it).
FVSR_DEV void outside(int p, int64_t rows, float (&cs)[8]) {
  const bool in = p >= 0 && p < rows;
#pragma unroll
  for (int e = 0; e < 8; e += 2) cs[e] = in ? cs[e] : __builtin_nanf("");
}

// cos and sin of dims d0..d0+7 of token t.
template <int D>
FVSR_DEV void load_turn(const Args& a, int t, int d0, float (&cs)[8]) {
  const int p = a.positions ? a.positions[t] : t;
  load8(a.cs, FVSR_DT_F32, (int64_t)(p >= 0 && p < a.cs_rows ? p : 0) * D + d0, cs);
  outside(p, a.cs_rows, cs);
}

// NaNs as they lie in memory may signal, of which v_max3_f32 would lose what it held.
FVSR_DEV void quieten(float (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = __builtin_canonicalizef(x[e]);
}

// x * r * w, then the rotation of its four pairs.
FVSR_DEV void norm_turn(float (&x)[8], bool norm, float r, const float (&w)[8], bool turn,
                        const float (&cs)[8]) {
  if (norm) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = x[e] * r * w[e];
  }
  if (turn) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float a = x[e], b = x[e + 1], c = cs[e], s = cs[e + 1];
      x[e] = __builtin_fmaf(a, c, -(b * s));
      x[e + 1] = __builtin_fmaf(a, s, b * c);
    }
  }
}

// The same in 64 bits (k): x * w is exact, its product with r rounded once.
FVSR_DEV void norm_turn64(float (&x)[8], bool norm, double r, const float (&w)[8], bool turn,
                          const float (&cs)[8]) {
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    double a = x[e], b = x[e + 1];
    if (norm) a = a * w[e] * r, b = b * w[e + 1] * r;
    if (turn) {
      const double c = cs[e], s = cs[e + 1], t = __builtin_fma(a, c, -(b * s));
      b = __builtin_fma(a, s, b * c);
      a = t;
    }
    if (norm || turn) x[e] = to_odd(a), x[e + 1] = to_odd(b);
  }
}

// q rows without a row norm: a thread per eight elements.
template <int DT, int D>
FVSR_DEV void q_chunk(const Args& a, int64_t chunk) {
  constexpr int C = D / 8;
  const int64_t unit = chunk / C;  // (token, head)
  const bool live = unit < (int64_t)a.T * a.q_heads;
  const int t = live ? (int)(unit / a.q_heads) : 0, h = live ? (int)(unit % a.q_heads) : 0;
  const int d0 = (int)(chunk % C) * 8;
  float x[8], w[8] = {}, cs[8] = {};
  load8(a.q, DT, t * a.q_ts + h * a.q_hs + d0, x);
  if (a.cs) load_turn<D>(a, t, d0, cs);
  float r = 1.0f;
  if (a.q_norm == kHead) {
    load8(a.q_weight, a.w_dt, d0, w);
    r = inv_rms(lanes_sum<C>(sum_sq<float>(x)), D, a.eps);
  }
  norm_turn(x, a.q_norm == kHead, r, w, a.cs != nullptr, cs);
  if (live) store8(a.q_out, DT, unit * D + d0, x);
}

// A q row with a norm over all of it: a wave per token.  (A lane's pieces are the
// same dims of their heads, so one load of cos and sin serves them all.)
template <int DT, int D, int N>
FVSR_DEV void q_row(const Args& a, int t) {
  if (t >= a.T) return;
  constexpr int C = D / 8;
  const int lane = threadIdx.x & 63, n = a.q_heads * C, d0 = lane % C * 8;
  float cs[8] = {};
  if (a.cs) load_turn<D>(a, t, d0, cs);
  Raw8<DT> held[N];
  const float r = inv_rms(load_row<float, DT, D>(a.q, t * a.q_ts, a.q_hs, a.q_heads, held),
                          a.q_heads * D, a.eps);
  const auto put = [&](float(&x)[8], int c) {
    float w[8];
    load8(a.q_weight, a.w_dt, c * 8, w);
    norm_turn(x, true, r, w, a.cs != nullptr, cs);
    store8(a.q_out, DT, (int64_t)t * n * 8 + c * 8, x);
  };
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float x[8];
    widen(held[i], x);
    if (lane + 64 * i < n) put(x, lane + 64 * i);
  }
  for (int c = lane + 64 * N; c < n; c += 64) {
    float x[8];
    load8(a.q, DT, t * a.q_ts + (c / C) * a.q_hs + d0, x);
    put(x, c);
  }
}

template <int DT, int D, int N>
FVSR_DEV void q_rows(const Args& a, int64_t wg) {
  if (a.q_norm == kRow)
    q_row<DT, D, N>(a, (int)(wg * (kWg<D> / 64) + (threadIdx.x >> 6)));
  else
    q_chunk<DT, D>(a, wg * kWg<D> + threadIdx.x);
}

// Scale exponent of a largest magnitude, given as its (finite) bits: 448 =
// 1.75 * 2^8, so a mantissa above 1.75 carries into the exponent.
FVSR_DEV int scale_exp(uint32_t top) { return max((int)((top + 0x1fffffu) >> 23) - 135, -126); }

FVSR_DEV float finite_abs(float x) {
  return fabsf(x) < __builtin_huge_valf() ? fabsf(x) : 0.0f;  // infinity, NaN: 0
}

// Four held codes at another scale: exact but for results below 2^-6.
FVSR_DEV uint32_t rescale4(uint32_t w, float f) {
  typedef float v2f __attribute__((ext_vector_type(2)));
  const v2f a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const v2f b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  return e4m3x4(a[0] * f, a[1] * f, b[0] * f, b[1] * f);
}

FVSR_DEV float pow2(int e) { return __builtin_ldexpf(1.0f, e); }

// Four values / f (a power of two) as e4m3; infinities and NaN give NaN.
FVSR_DEV uint32_t codes4(float a, float b, float c, float d, float f) {
  typedef short v2s __attribute__((ext_vector_type(2)));
  v2s t = {};
  t = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(t, a, b, f, false);
  t = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(t, c, d, f, true);
  return __builtin_bit_cast(uint32_t, t);
}

// A page's new tokens: slots lo .. hi - 1, slot 0 being row row0 of the call.  The page id
// is looked at only once the rows are on their way: it is one load more to wait for.
struct Job {
  int lo, hi, row0, h;
  int64_t id;
  __device__ __forceinline__ bool there(const Args& a) const { return id >= 0 && id < a.c.pages; }
  __device__ __forceinline__ int64_t ph(const Args& a) const { return id * a.c.heads + h; }
};

// The largest of all threads' magnitudes (not NaN), as bits.  An infinity among
// them: once more over the finite ones, of which again() gives a thread's largest.
template <int W, class Again>
FVSR_DEV uint32_t page_top(float top, float (&lds)[W], Again again) {
  const auto reduce = [&](float t) {
    t = wave_max_abs(t);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = t;
    __syncthreads();
    float m = lds[0];
#pragma unroll
    for (int w = 1; w < W; ++w) m = fmaxf(m, lds[w]);
    return m;
  };
  top = reduce(top);
  if (__builtin_isinf(top)) {
    __syncthreads();
    top = reduce(again());
  }
  return __float_as_uint(top);
}

// Runs body(full): true if every slot of the page is new and its rows can load
// together, else with a test of each row.
template <class Body>
FVSR_DEV void rows_of(const Job& j, Body body) {
  if (j.lo == 0 && j.hi == kPage)
    body(std::true_type{});
  else
    body(std::false_type{});
}

template <int DT, int D>
FVSR_DEV void append_k(const Args& a, const Job& j, double (&stat)[kPage],
                       float (&tops)[kWg<D> / 64]) {
  constexpr int C = D / 8, R = kTokens;
  const int tid = threadIdx.x, H = (int)a.c.heads;
  uint8_t* const scale = (uint8_t*)a.c.k_scale;
  int held = 0;
  // Row norms that no launch before has summed: a wave per token.
  if (a.k_norm == kRow && !a.row_stat) {
    for (int i = j.lo + (tid >> 6); i < j.hi; i += kWg<D> / 64) {
      const double r =
          inv_rms64(row_sq<DT, D, 1>(a.k, (j.row0 + i) * a.k_ts, a.k_hs, H), a.k_per, a.eps);
      if ((tid & 63) == 0) stat[i] = r;
    }
    __syncthreads();
  }
  const int d0 = (tid % C) * 8, slot0 = tid / C * R;
  float w[8] = {};
  if (a.k_norm != kNone) load8(a.k_weight, a.w_dt, (a.k_norm == kRow ? j.h * D : 0) + d0, w);
  float x[R][8];
  float top = 0.0f;
  uint32_t near = 0;  // bit i: a value of token i is near a border
  rows_of(j, [&](auto full) {
    const auto live = [&](int i) { return full || (slot0 + i >= j.lo && slot0 + i < j.hi); };
    // All positions and rows go out together, then the rotations: not one load behind
    // another for each of the four tokens.
    Raw8<DT> raw[R];
    constexpr int Q = D == 64 ? 1 : 2;  // rotations in flight (registers)
    Raw8<FVSR_DT_F32> turn[Q];
    int pos[R];
    float rs[R] = {};
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int t = j.row0 + (live(i) ? slot0 + i : j.lo);
      pos[i] = a.positions ? a.positions[t] : t;
      if (a.k_norm == kRow) rs[i] = (float)(a.row_stat ? a.row_stat[t] : stat[t - j.row0]);
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      raw[i] = Raw8<DT>{};
      if (live(i))
        raw[i] = load_raw<DT>(a.k, (int64_t)(j.row0 + slot0 + i) * a.k_ts + j.h * a.k_hs + d0);
    }
    if (j.there(a)) held = scale[j.ph(a)];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (a.cs && i % Q == 0) {
#pragma unroll
        for (int k = 0; k < Q; ++k) {
          const int p = pos[i + k];
          turn[k] = load_raw<FVSR_DT_F32>(
              a.cs, (int64_t)(p >= 0 && p < a.cs_rows ? p : 0) * D + d0);
        }
      }
      widen(raw[i], x[i]);
      if (!full && __ballot(live(i)) == 0) continue;
      float cs[8] = {};
      if (a.cs) {
        widen(turn[i % Q], cs);
        outside(pos[i], a.cs_rows, cs);
      }
      float r = 1.0f;
      if (a.k_norm == kHead)
        r = (float)inv_rms64(lanes_sum<C>(sum_sq<double>(x[i])), a.k_per, a.eps);
      if (a.k_norm == kRow) r = rs[i];
      norm_turn(x[i], a.k_norm != kNone, r, w, a.cs != nullptr, cs);
      if (a.k_norm == kNone && !a.cs) quieten(x[i]);
      if (!live(i)) continue;
      Border b;
#pragma unroll
      for (int e = 0; e < 8; ++e) b.see(x[i][e]);
      near |= (uint32_t)b.near() << i;
#pragma unroll
      for (int e = 0; e < 8; e += 2) top = max3_abs(top, x[i][e], x[i][e + 1]);
    }
  });
  if (!j.there(a)) return;  // no such page: dropped
  int e = scale_exp(page_top(top, tops, [&] {
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (slot0 + i >= j.lo && slot0 + i < j.hi) t = fmaxf(t, finite_abs(x[i][k]));
    return t;
  }));
  const int old = held - 127;
  if (j.lo > 0) e = max(e, old);
  if (tid == 0) scale[j.ph(a)] = (uint8_t)(e + 127);
  uint8_t* const page = (uint8_t*)a.c.k + j.ph(a) * kPage * D;
  const float f = pow2(e);
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int slot = slot0 + i;
    u32x2_t* const p = (u32x2_t*)(page + slot * D + d0);
    if (slot >= j.lo && slot < j.hi) {
      *p = u32x2_t{codes4(x[i][0], x[i][1], x[i][2], x[i][3], f),
                   codes4(x[i][4], x[i][5], x[i][6], x[i][7], f)};
    } else if (slot < j.lo && e != old) {
      const u32x2_t c = *p;
      *p = u32x2_t{rescale4(c[0], pow2(old - e)), rescale4(c[1], pow2(old - e))};
    }
  }
  if (__ballot(near) == 0 || (a.k_norm == kNone && !a.cs)) return;
  // Tokens near a border, by now with the registers free.
#pragma unroll 1
  for (int i = 0; i < R; ++i) {
    if (__ballot(near >> i & 1) == 0) continue;
    const int slot = min(max(slot0 + i, j.lo), j.hi - 1), t = j.row0 + slot;
    float y[8], cs[8] = {};
    widen(load_raw<DT>(a.k, (int64_t)t * a.k_ts + j.h * a.k_hs + d0), y);
    if (a.cs) load_turn<D>(a, t, d0, cs);
    if (a.k_norm != kNone) load8(a.k_weight, a.w_dt, (a.k_norm == kRow ? j.h * D : 0) + d0, w);
    double r = 1.0;
    if (a.k_norm == kHead) r = inv_rms64(lanes_sum<C>(sum_sq<double>(y)), a.k_per, a.eps);
    if (a.k_norm == kRow) r = a.row_stat ? a.row_stat[t] : stat[slot];
    norm_turn64(y, a.k_norm != kNone, r, w, a.cs != nullptr, cs);
    if (slot == slot0 + i)
      *(u32x2_t*)(page + slot * D + d0) = u32x2_t{codes4(y[0], y[1], y[2], y[3], f),
                                                  codes4(y[4], y[5], y[6], y[7], f)};
  }
}

template <int DT, int D>
FVSR_DEV void append_v(const Args& a, const Job& j, uint8_t* vt, float (&tops)[kWg<D> / 64]) {
  constexpr int C = D / 8, R = kTokens;
  const int tid = threadIdx.x;
  uint8_t* const scale = (uint8_t*)a.c.v_scale;
  const int d0 = (tid % C) * 8, slot0 = tid / C * R;
  Raw8<DT> raw[R];
  float top = 0.0f;
  rows_of(j, [&](auto full) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      raw[i] = Raw8<DT>{};
      if (full || (slot0 + i >= j.lo && slot0 + i < j.hi))
        raw[i] = load_raw<DT>(a.v, (int64_t)(j.row0 + slot0 + i) * a.v_ts + j.h * a.v_hs + d0);
    }
  });
  if (!j.there(a)) return;  // no such page: dropped
  const int held = scale[j.ph(a)];  // (its use waits for it: after the rows)
#pragma unroll
  for (int i = 0; i < R; ++i) {
    float y[8];
    widen(raw[i], y);
    if constexpr (DT != FVSR_DT_F16) quieten(y);  // (fp16: its conversion did)
#pragma unroll
    for (int k = 0; k < 8; k += 2) top = max3_abs(top, y[k], y[k + 1]);
  }
  int e = scale_exp(page_top(top, tops, [&] {
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float y[8];
      widen(raw[i], y);
#pragma unroll
      for (int k = 0; k < 8; ++k) t = fmaxf(t, finite_abs(y[k]));
    }
    return t;
  }));
  const int old = held - 127;
  if (j.lo > 0) e = max(e, old);
  if (tid == 0) scale[j.ph(a)] = (uint8_t)(e + 127);
  // [dim][token]: a thread's R tokens of a dim are one unit of R bytes; unit u
  // of row d sits at u ^ (d / 8 % 16), so that the D/8 threads of a token spread
  // over the banks.
  const auto vt_at = [&](int d, int u) { return vt + d * kPage + (u ^ ((d >> 3) & 15)) * R; };
  const float f = pow2(e);
#pragma unroll
  for (int g = 0; g < R / 4; ++g) {
    float y[4][8];
#pragma unroll
    for (int i = 0; i < 4; ++i) widen(raw[4 * g + i], y[i]);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      *(uint32_t*)(vt_at(d0 + k, slot0 / R) + 4 * g) =
          codes4(y[0][k], y[1][k], y[2][k], y[3][k], f);
  }
  __syncthreads();
  uint8_t* const page = (uint8_t*)a.c.v + j.ph(a) * kPage * D;
  const auto piece = [&](int d, int s0) {  // 16 tokens' codes of a dim
    u32x4_t c;
#pragma unroll
    for (int g = 0; g < 16 / R; ++g)
      __builtin_memcpy((uint8_t*)&c + g * R,
                       __builtin_assume_aligned(vt_at(d, s0 / R + g), R), R);
    return c;
  };
  constexpr int P = kPage / 16;  // pieces of a dim
  if (j.lo == 0 && j.hi == kPage) {
#pragma unroll
    for (int it = 0; it < D * P / kWg<D>; ++it) {
      const int idx = it * kWg<D> + tid, d = idx / P, s0 = idx % P * 16;
      *(u32x4_t*)(page + d * kPage + s0) = piece(d, s0);
    }
    return;
  }
#pragma unroll 1
  for (int idx = tid; idx < D * P; idx += kWg<D>) {
    const int d = idx / P, s0 = idx % P * 16;
    const bool grow = s0 < j.lo && e != old;  // held codes to round again
    if ((s0 + 16 <= j.lo && !grow) || s0 >= j.hi) continue;
    uint8_t* const p = page + d * kPage + s0;
    if (s0 >= j.lo && s0 + 16 <= j.hi) {
      *(u32x4_t*)p = piece(d, s0);
    } else if (grow) {
      const u32x4_t c = piece(d, s0);
      u32x4_t o = *(const u32x4_t*)p;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const uint32_t n = rescale4(o[g], pow2(old - e));
        uint32_t m = 0, keep = 0;  // bytes of new tokens; bytes behind them
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int slot = s0 + 4 * g + k;
          if (slot >= j.hi) keep |= 0xffu << (8 * k);
          else if (slot >= j.lo) m |= 0xffu << (8 * k);
        }
        o[g] = (c[g] & m) | (o[g] & keep) | (n & ~(m | keep));
      }
      *(u32x4_t*)p = o;
    } else {
#pragma unroll 1
      for (int k = max(j.lo - s0, 0); k < min(j.hi - s0, 16); ++k)
        p[k] = vt_at(d, (s0 + k) / R)[(s0 + k) % R];
    }
  }
}

// Workgroup wg's part of a page: units * heads workgroups, for k and v each if both.
enum { kKeys = 1, kValues = 2 };
template <int DT, int D, int KINDS>
FVSR_DEV void page_part(const Args& a, int wg) {
  constexpr int n = KINDS == (kKeys | kValues) ? 2 : 1;
  // A page's heads share the rotations of its tokens: they take one XCD's
  // L2 (workgroups go round robin over the 8).
  const int H = (int)a.c.heads, turn = wg / 8;
  const int part = turn % (n * H), unit = turn / (n * H) * 8 + wg % 8;
  if (unit >= a.units) return;

  SeqPart s;
  const auto pages_of = [](int n, int len) {
    const int at = max(len - n, 0);
    return len > at ? (len - 1) / kPage - at / kPage + 1 : 0;
  };
  if (a.c.cu) {
    if (!find_part(a.c.cu, a.c.lengths, (int)a.c.sequences, a.T, unit, false, pages_of, s)) return;
  } else {
    s.b = unit / a.units_max;
    s.part = unit % a.units_max;
    s.rows = seq_rows(nullptr, s.b, (int)a.c.sequences, a.T);
    s.len = max(a.c.lengths[s.b], 0);
    if (s.part >= pages_of(s.rows.n, s.len)) return;
  }
  const int at = s.len - s.rows.n;          // position of the sequence's first new token
  const int page = max(at, 0) / kPage + s.part;
  if (page >= a.c.table_pages) return;      // past the table: dropped
  Job j;
  j.id = a.c.table[s.b * a.c.table_stride + page];
  j.lo = max(max(at, 0), page * kPage) - page * kPage;
  j.hi = min(s.len - page * kPage, kPage);
  j.row0 = s.rows.lo + page * kPage - at;
  j.h = part / n;
  __shared__ float tops[kWg<D> / 64];
  if constexpr ((KINDS & kValues) != 0) {
    __shared__ __attribute__((aligned(16))) uint8_t vt[D * kPage];  // v's codes, [dim][token]
    if (n == 1 || part % n) return append_v<DT, D>(a, j, vt, tops);
  }
  if constexpr ((KINDS & kKeys) != 0) {
    __shared__ double stat[kPage];
    append_k<DT, D>(a, j, stat, tops);
  }
}

template <int DT, int D>
__global__ __launch_bounds__(kWg<D>) void kv_append_kernel(Args a) {
  if ((int)blockIdx.x < a.page_wgs)
    page_part<DT, D, kKeys | kValues>(a, blockIdx.x);
  else
    q_rows<DT, D, 1>(a, blockIdx.x - a.page_wgs);
}

// Row norms of many tokens take two launches: v beside the k statistics, then the q
// rows and k, read again.  (The q rows first or last: 16896 tokens x 12 heads 73.2 us, 72.2.)

// Pieces of a row that its wave holds: rows of 2048 elements.  Eight take registers from the
// pages of the launch (16896 tokens x 12 heads 73.4 us, 80.2 with eight; one prompt of 2000 x 32
// heads 25.6, 27.7) and save a second read of longer q rows (8 prompts of 2000 x 32/8 heads 107
// us, 102 with eight).
constexpr int kHeld = 4;
template <int DT, int D>
__global__ __launch_bounds__(kWg<D>) void kv_rows_kernel(Args a) {
  constexpr int W = kWg<D> / 64;
  if ((int)blockIdx.x < a.page_wgs) return page_part<DT, D, kValues>(a, blockIdx.x);
  const int t = ((int)blockIdx.x - a.page_wgs) * W + (threadIdx.x >> 6);
  if (t >= a.T) return;
  const int H = (int)a.c.heads;
  const double r = inv_rms64(row_sq<DT, D, kHeld>(a.k, t * a.k_ts, a.k_hs, H), a.k_per, a.eps);
  if ((threadIdx.x & 63) == 0) a.row_stat[t] = r;
}

template <int DT, int D>
__global__ __launch_bounds__(kWg<D>) void kv_keys_kernel(Args a) {
  const int q_wgs = gridDim.x - a.page_wgs;
  if ((int)blockIdx.x < q_wgs)
    q_rows<DT, D, kHeld>(a, blockIdx.x);
  else
    page_part<DT, D, kKeys>(a, blockIdx.x - q_wgs);
}

// Two neighbouring elements as fp32.
template <int DT>
FVSR_DEV void load2(const void* p, int64_t i, float (&x)[2]) {
  if constexpr (DT == FVSR_DT_F32) {
    const float* s = (const float*)p + i;
    x[0] = s[0], x[1] = s[1];
  } else {
    const uint32_t u = *(const uint32_t*)((const uint16_t*)p + i);
    if constexpr (DT == FVSR_DT_F16) {
      x[0] = (float)__builtin_bit_cast(_Float16, (uint16_t)u);
      x[1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(u >> 16));
    } else {
      x[0] = bf_lo(u), x[1] = bf_hi(u);
    }
  }
}

FVSR_DEV float fused(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
FVSR_DEV double fused(double a, double b, double c) { return __builtin_fma(a, b, c); }

// Norm and rotation of two dims d0, d0 + 1 of a head of N tokens t in F, a wave per head;
// `ts`, `hs` and `heads` describe the rows of src (q or k).  Each kind of load goes out
// for all tokens at once.  Sums are in S, but a row's of eight squares at a time in F: all
// of it in 64 bits takes 64 x 5 tokens with row norms from 18.8 to 22.6 us.
template <class F, class S, int DT, int D, int N>
FVSR_DEV void turn2(const Args& a, const void* src, int64_t ts, int64_t hs, int heads,
                    const void* weight, int norm, const int (&t)[N], int h, int d0,
                    float (&x)[N][2]) {
  const int lane = threadIdx.x & 63;
  int pos[N];
#pragma unroll
  for (int i = 0; i < N; ++i) pos[i] = a.positions ? a.positions[t[i]] : t[i];
  S sq[N] = {};
  float cs[N][2];
  if (norm == kRow) {
    for (int c = lane; c < heads * (D / 8); c += 64) {
      const int64_t at = (c / (D / 8)) * hs + (c % (D / 8)) * 8;
      Raw8<DT> raw[N];
#pragma unroll
      for (int i = 0; i < N; ++i) raw[i] = load_raw<DT>(src, t[i] * ts + at);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float r[8];
        widen(raw[i], r);
        sq[i] += (S)sum_sq<F>(r);
      }
    }
  } else if (norm == kHead) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      sq[i] = lane * 2 < D ? (S)x[i][0] * (S)x[i][0] + (S)x[i][1] * (S)x[i][1] : (S)0;
  }
  if (a.cs) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const bool in = pos[i] >= 0 && pos[i] < a.cs_rows;
      const float* p = a.cs + (int64_t)(in ? pos[i] : 0) * D + d0;
      cs[i][0] = in ? p[0] : __builtin_nanf("");
      cs[i][1] = p[1];
    }
  }
  if (norm == kNone && !a.cs) return;
  float w[2] = {1.0f, 1.0f};
  if (norm != kNone) {
#pragma unroll
    for (int e = 0; e < 2; ++e)
      w[e] = ld_elem(weight, a.w_dt, (norm == kRow ? h * D : 0) + d0 + e);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    F u = x[i][0], v = x[i][1];
    if (norm != kNone) {
      F r;
      S sum = lanes_sum<64>(sq[i]);
      if constexpr (std::is_same_v<S, double>) {
        // (Squares that fp32 does not hold: rare, and the same for the whole wave.)
        if (std::is_same_v<F, float> && norm == kRow && !(sum > 0x1p-80 && sum < 0x1p127))
          sum = row_sq<DT, D, 1>(src, t[i] * ts, hs, heads);
        r = (F)inv_rms64(sum, a.k_per, a.eps);
      } else {
        r = inv_rms(sum, norm == kRow ? heads * D : D, a.eps);
      }
      if constexpr (std::is_same_v<F, double>)
        u = u * w[0] * r, v = v * w[1] * r;  // (x * w is exact)
      else
        u = u * r * w[0], v = v * r * w[1];  // (x * w may be more than fp32 holds)
    }
    if (a.cs) {
      const F c = cs[i][0], s = cs[i][1], o = fused(u, c, -(v * s));
      v = fused(u, s, v * c);
      u = o;
    }
    if constexpr (std::is_same_v<F, double>)
      x[i][0] = to_odd(u), x[i][1] = to_odd(v);
    else
      x[i][0] = u, x[i][1] = v;
  }
}

// The step of at most N tokens per sequence, the same number for each: a wave per
// (page of a sequence, head), of k and v, or per q head of a token; two dims a lane (64
// dims: the upper lanes repeat the lower ones).  It is all latency: one token's row, lengths
// and positions load at once, then the page id and the rotation, then the page's
// scales; a norm over the row is summed by every wave for itself.  A page whose scale
// grows (rare: a power of two) has its held codes rounded again by the wave.  64 x 5 tokens,
// 32 / 8 heads: 16.6 us by pages as a prompt's, 9.6 so (row norms: 21.7, 18.8); 64 x 8 17.7, 12.9.
template <int DT, int D, int N>
__global__ __launch_bounds__(kThreads) void kv_token_kernel(Args a) {
  const int lane = threadIdx.x & 63, d0 = lane * 2 % D;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr int parts = N == 1 ? 1 : 2;  // pages that a sequence's tokens can touch
  const int H = (int)a.c.heads, unit = blockIdx.x * 4 + wave;
  const int B = (int)a.c.sequences, kv_units = B * parts * H;
  if (unit >= kv_units + a.T * a.q_heads) return;
  if (unit >= kv_units) {
    const int u = unit - kv_units, t[1] = {u / a.q_heads}, h = u % a.q_heads;
    float xs[1][2];
    float(&x)[2] = xs[0];
    load2<DT>(a.q, t[0] * a.q_ts + h * a.q_hs + d0, x);
    turn2<float, float, DT, D, 1>(a, a.q, a.q_ts, a.q_hs, a.q_heads, a.q_weight, a.q_norm, t, h,
                                  d0, xs);
    if (lane * 2 >= D) return;
    const int64_t o = (int64_t)u * D + d0;
    if constexpr (DT == FVSR_DT_F32) {
      ((float*)a.q_out)[o] = x[0], ((float*)a.q_out)[o + 1] = x[1];
    } else {
      const uint32_t c = DT == FVSR_DT_F16
                             ? (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)x[0]) |
                                   (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)x[1]) << 16
                             : pack_bf16x2(x[0], x[1]);
      *(uint32_t*)((uint16_t*)a.q_out + o) = c;
    }
    return;
  }
  const int b = unit / H / parts, part = unit / H % parts, h = unit % H;
  const int n = N == 1 ? 1 : a.T / B, len = max(a.c.lengths[b], 0), at = len - n;
  const int page = max(at, 0) / kPage + part;
  if (N > 1 && page > max(len - 1, 0) / kPage) return;  // (its positions may pass 32 bits)
  const int lo = max(max(at, 0), page * kPage) - page * kPage, hi = min(len - page * kPage, kPage);
  if (N > 1 && hi <= lo) return;
  // Tokens of slots lo .. hi - 1, the last one repeated.
  int t[N];
#pragma unroll
  for (int i = 0; i < N; ++i)
    t[i] = N == 1 ? b : b * n + page * kPage - at + lo + min(i, hi - lo - 1);
  float x[N][2], y[N][2], kt = 0.0f, vt = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    load2<DT>(a.k, t[i] * a.k_ts + h * a.k_hs + d0, x[i]);
    load2<DT>(a.v, t[i] * a.v_ts + h * a.v_hs + d0, y[i]);
  }
  turn2<float, double, DT, D, N>(a, a.k, a.k_ts, a.k_hs, H, a.k_weight, a.k_norm, t, h, d0, x);
  uint32_t near = 0;  // bit i: a value of token i is near a border
#pragma unroll
  for (int i = 0; i < N; ++i) {
    Border b;
    b.see(x[i][0]), b.see(x[i][1]);
    near |= (uint32_t)b.near() << i;
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e)
      kt = fmaxf(kt, finite_abs(x[i][e])), vt = fmaxf(vt, finite_abs(y[i][e]));
  if (hi <= lo || page >= a.c.table_pages) return;
  const int64_t id = __builtin_amdgcn_readfirstlane(a.c.table[b * a.c.table_stride + page]);
  if (id < 0 || id >= a.c.pages) return;
  const int64_t ph = id * H + h;
  uint8_t* const ksp = (uint8_t*)a.c.k_scale + ph;
  uint8_t* const vsp = (uint8_t*)a.c.v_scale + ph;
  const int k_old = *ksp - 127, v_old = *vsp - 127;
  int ke = scale_exp(__float_as_uint(wave_max_abs(kt)));
  int ve = scale_exp(__float_as_uint(wave_max_abs(vt)));
  if (lo > 0) ke = max(ke, k_old), ve = max(ve, v_old);
  uint8_t* const kp = (uint8_t*)a.c.k + ph * kPage * D;
  uint8_t* const vp = (uint8_t*)a.c.v + ph * kPage * D;
  if (lo > 0 && (ke != k_old || ve != v_old)) {
    if (ke != k_old) {
      const float f = pow2(k_old - ke);
      for (int c = lane; c < lo * (D / 16); c += 64) {
        u32x4_t* const p = (u32x4_t*)(kp + c * 16);
        u32x4_t o = *p;
#pragma unroll
        for (int g = 0; g < 4; ++g) o[g] = rescale4(o[g], f);
        *p = o;
      }
    }
    if (ve != v_old) {
      const float f = pow2(v_old - ve);
      const int per = (lo + 15) / 16;  // pieces of a dim with held tokens
      for (int c = lane; c < D * per; c += 64) {
        const int s0 = c % per * 16;
        u32x4_t* const p = (u32x4_t*)(vp + c / per * kPage + s0);
        u32x4_t o = *p;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int held = min(max(lo - s0 - 4 * g, 0), 4);  // of these four
          const uint32_t m = held == 4 ? ~0u : (1u << (8 * held)) - 1;
          o[g] = (rescale4(o[g], f) & m) | (o[g] & ~m);
        }
        *p = o;
      }
    }
    __builtin_amdgcn_s_waitcnt(0);  // before the new tokens go into the same pieces
  }
  const auto put_k = [&](int slot, const float(&x)[2]) {
    *(uint16_t*)(kp + slot * D + d0) = (uint16_t)codes4(x[0], x[1], 0.0f, 0.0f, pow2(ke));
  };
  const bool both = lane * 2 < D;  // (the upper lanes of 64 dims store nothing)
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if ((N > 1 && i >= hi - lo) || !both) continue;
    const int slot = lo + i;
    put_k(slot, x[i]);
    const uint32_t c = codes4(y[i][0], y[i][1], 0.0f, 0.0f, pow2(ve));
    vp[d0 * kPage + slot] = (uint8_t)c;
    vp[(d0 + 1) * kPage + slot] = (uint8_t)(c >> 8);
  }
  if (lane == 0) *ksp = (uint8_t)(ke + 127), *vsp = (uint8_t)(ve + 127);
  if (__ballot(near) == 0 || (a.k_norm == kNone && !a.cs)) return;
#pragma unroll 1
  for (int i = 0; i < min(N, hi - lo); ++i) {
    if (__ballot(near >> i & 1) == 0) continue;
    const int one[1] = {N == 1 ? b : b * n + page * kPage - at + lo + i};
    float y[1][2];
    load2<DT>(a.k, one[0] * a.k_ts + h * a.k_hs + d0, y[0]);
    turn2<double, double, DT, D, 1>(a, a.k, a.k_ts, a.k_hs, H, a.k_weight, a.k_norm, one, h, d0, y);
    if (both) put_k(lo + i, y[0]);
  }
}

constexpr int kFew = 8;  // tokens per sequence that a wave takes

// Tokens up to which each workgroup sums its own rows for a row norm.
constexpr int64_t kOwnStat = 64;

template <int DT, int D>
void launch(const Args& a, int64_t units, hipStream_t st) {
  if (!a.c.cu && a.T <= kFew * a.c.sequences) {
    const bool one = a.T == a.c.sequences;
    const int64_t waves = (one ? 1 : 2) * a.c.sequences * a.c.heads + (int64_t)a.T * a.q_heads;
    const auto kernel = one ? kv_token_kernel<DT, D, 1> : kv_token_kernel<DT, D, kFew>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)((waves + 3) / 4)), dim3(kThreads), 0, st, a);
    return;
  }
  Args b = a;
  b.units = (int)units;
  b.page_wgs = (int)((units + 7) / 8 * 8 * a.c.heads) * (a.row_stat ? 1 : 2);
  constexpr int W = kWg<D> / 64;
  const int64_t q_wgs =
      !a.q                ? 0
      : a.q_norm == kRow ? (a.T + W - 1) / W
                         : ((int64_t)a.T * a.q_heads * (D / 8) + kWg<D> - 1) / kWg<D>;
  const dim3 block(kWg<D>);
  if (a.row_stat) {
    hipLaunchKernelGGL((kv_rows_kernel<DT, D>),
                       dim3((unsigned)(b.page_wgs + (a.T + W - 1) / W)), block, 0, st, b);
    hipLaunchKernelGGL((kv_keys_kernel<DT, D>), dim3((unsigned)(b.page_wgs + q_wgs)), block, 0, st,
                       b);
  } else {
    hipLaunchKernelGGL((kv_append_kernel<DT, D>), dim3((unsigned)(b.page_wgs + q_wgs)), block, 0,
                       st, b);
  }
}

bool rows_aligned(const void* p, int64_t ts, int64_t hs, int64_t size) {
  return (((uintptr_t)p | (uint64_t)(ts * size) | (uint64_t)(hs * size)) & 15) == 0;
}

}  // namespace

extern "C" int64_t fvsr_kv_append_workspace_floats(int64_t T, int k_norm) {
  return k_norm == FVSR_NORM_ROW && T > kOwnStat && T <= kMaxRows ? 2 * T : 0;
}

extern "C" int fvsr_kv_append(const fvsr_kv_cache* cache, const void* k, int64_t k_tok_stride,
                              int64_t k_head_stride, const void* v, int64_t v_tok_stride,
                              int64_t v_head_stride, const void* q, int64_t q_tok_stride,
                              int64_t q_head_stride, int64_t q_heads, void* q_out, int dtype,
                              int64_t T, const void* k_weight, int k_norm, const void* q_weight,
                              int q_norm, int weight_dtype, float eps, const float* cs,
                              int64_t cs_rows, const int32_t* positions, float* workspace,
                              int64_t workspace_floats, void* stream) {
  int rc = kv_cache_ok(cache, T);
  if (rc != FVSR_OK) return rc;
  if (dtype < 0 || dtype > FVSR_DT_F32 || weight_dtype < 0 || weight_dtype > FVSR_DT_F32 ||
      k_norm < 0 || k_norm > FVSR_NORM_ROW || q_norm < 0 || q_norm > FVSR_NORM_ROW)
    return FVSR_EINVAL;
  if (q && (q_heads <= 0 || !q_out)) return FVSR_EINVAL;
  if (q && q_heads > kMaxBlocks) return FVSR_EUNSUPPORTED;
  if ((k_norm && !k_weight) || (q && q_norm && !q_weight)) return FVSR_EINVAL;
  if (cs && (cs_rows <= 0 || (!positions && cs_rows < T))) return FVSR_EINVAL;
  const int64_t size = dtype == FVSR_DT_F32 ? 4 : 2, D = cache->head_dim, B = cache->sequences;
  // Without sequences no row of k and v has a place, but the q rows are turned.
  if (T == 0 || (B == 0 && !q)) return FVSR_OK;
  if (B > 0 && (!k || !v)) return FVSR_EINVAL;
  if ((B > 0 && (!rows_aligned(k, k_tok_stride, k_head_stride, size) ||
                 !rows_aligned(v, v_tok_stride, v_head_stride, size))) ||
      (q && !rows_aligned(q, q_tok_stride, q_head_stride, size)) ||
      (((uintptr_t)q_out | (uintptr_t)k_weight | (uintptr_t)q_weight | (uintptr_t)cs) & 15))
    return FVSR_EUNSUPPORTED;
  const int64_t need = B > 0 ? fvsr_kv_append_workspace_floats(T, k_norm) : 0;
  if (need && (!workspace || workspace_floats < need)) return FVSR_EWORKSPACE;
  if (need && ((uintptr_t)workspace & 7)) return FVSR_EUNSUPPORTED;
  // Pages that n tokens touch: at most n, and at most (n + 126) / 128 + 1.
  const auto most = [](int64_t n) { return std::min(n, (n + 126) / kPage + 1); };
  Args a{};
  a.c = *cache;
  a.k = k, a.v = v, a.q = q, a.k_weight = k_weight, a.q_weight = q_weight, a.q_out = q_out;
  a.cs = cs, a.positions = positions, a.row_stat = need ? (double*)workspace : nullptr;
  a.k_ts = k_tok_stride, a.k_hs = k_head_stride, a.v_ts = v_tok_stride, a.v_hs = v_head_stride;
  a.q_ts = q_tok_stride, a.q_hs = q_head_stride, a.cs_rows = cs_rows;
  a.T = (int)T, a.q_heads = q ? (int)q_heads : 0, a.k_norm = k_norm, a.q_norm = q_norm;
  a.w_dt = weight_dtype, a.eps = eps;
  a.k_per = 1.0 / (double)(k_norm == kRow ? cache->heads * D : D);
  a.units_max = B > 0 ? (int)most(T / B) : 0;
  // Packed rows: the sum of those bounds over any B counts that add up to T.
  const int64_t units = B > 0 && cache->cu ? std::min(T, (T + 126 * B) / kPage + B)
                                           : B * a.units_max;
  // Workgroups of either form of a launch, of 256 threads or twice that (kWg).
  const int64_t q_wgs = q ? T * q_heads / 4 + T / 4 + 2 : 0;
  if ((units + 7) * 2 * cache->heads + q_wgs > kMaxBlocks / 2 ||
      T * (cache->heads + a.q_heads) > kMaxBlocks * 64)
    return FVSR_EUNSUPPORTED;
  const hipStream_t st = (hipStream_t)stream;
  if (D == 128) {
    if (dtype == FVSR_DT_BF16) launch<FVSR_DT_BF16, 128>(a, units, st);
    if (dtype == FVSR_DT_F16) launch<FVSR_DT_F16, 128>(a, units, st);
    if (dtype == FVSR_DT_F32) launch<FVSR_DT_F32, 128>(a, units, st);
  } else {
    if (dtype == FVSR_DT_BF16) launch<FVSR_DT_BF16, 64>(a, units, st);
    if (dtype == FVSR_DT_F16) launch<FVSR_DT_F16, 64>(a, units, st);
    if (dtype == FVSR_DT_F32) launch<FVSR_DT_F32, 64>(a, units, st);
  }
  return fvsr_launch_status();
}
