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
// One workgroup per (page, head): a page's scale needs all of its new tokens at
// once, and 128 x 128 values of k and v fit its registers, so k and v are read
// once.  Thread t holds dims 8*(t % (D/8)).. of R consecutive tokens; v's codes
// turn to [dim][token] through LDS.  The q rows are further workgroups of the
// same launch.  An RMSNorm over whole rows needs other heads' values: the rows'
// statistics come from a launch before (which also does q), or, for a few
// tokens, each workgroup sums its own rows.
#include <algorithm>

#include "kv_pages.h"

namespace {

constexpr int kThreads = 256;
enum { kNone = FVSR_NORM_NONE, kHead = FVSR_NORM_HEAD, kRow = FVSR_NORM_ROW };

struct Args {
  fvsr_kv_cache c;
  const void *k, *v, *q, *k_weight, *q_weight;
  void* q_out;
  const float* cs;           // [cs_rows][D/2][2] (cos, sin); null: no rotation
  const int32_t* positions;  // row of cs for each token; null: the token's own number
  float* row_stat;           // 1/rms of each k row (row norm, from the launch before)
  int64_t k_ts, k_hs, v_ts, v_hs, q_ts, q_hs, cs_rows;
  int T, q_heads, k_norm, q_norm, w_dt, units_max, page_wgs;
  float eps;
};

// Eight consecutive elements as fp32 (16-byte aligned).
FVSR_DEV void load8(const void* p, int dt, int64_t i, float (&x)[8]) {
  if (dt == FVSR_DT_F32) {
    const f32x4_t* s = (const f32x4_t*)((const float*)p + i);
    const f32x4_t a = s[0], b = s[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = a[e], x[4 + e] = b[e];
  } else if (dt == FVSR_DT_F16) {
    typedef _Float16 h8 __attribute__((ext_vector_type(8)));
    const h8 a = *(const h8*)((const _Float16*)p + i);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)a[e];
  } else {
    const u32x4_t a = *(const u32x4_t*)((const uint16_t*)p + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[2 * e] = bf_lo(a[e]), x[2 * e + 1] = bf_hi(a[e]);
  }
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

FVSR_DEV float sum_sq(const float (&x)[8]) {
  float s = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) s = __builtin_fmaf(x[e], x[e], s);
  return s;
}

FVSR_DEV float inv_rms(float sq, int n, float eps) { return 1.0f / __builtin_sqrtf(sq / n + eps); }

// Sum over the D/8 lanes that hold one head.
template <int C>
FVSR_DEV float head_sum(float v) {
#pragma unroll
  for (int d = 1; d < C; d *= 2) v += __shfl_xor(v, d);
  return v;
}

// Sum of squares of a whole row of H heads by one wave.
template <int DT, int D>
FVSR_DEV float row_sq(const void* x, int64_t row, int64_t hs, int H) {
  const int lane = threadIdx.x & 63;
  float s = 0.0f;
  for (int c = lane; c < H * (D / 8); c += 64) {
    float a[8];
    load8(x, DT, row + (c / (D / 8)) * hs + (c % (D / 8)) * 8, a);
    s += sum_sq(a);
  }
  return wave_sum(s);
}

// cos and sin of dims d0..d0+7 of token t.  A position outside the table
// gives NaN instead of a read outside it.
template <int D>
FVSR_DEV void load_turn(const Args& a, int t, int d0, float (&cs)[8]) {
  const int64_t p = a.positions ? (int64_t)a.positions[t] : t;
  const bool in = p >= 0 && p < a.cs_rows;
  load8(a.cs, FVSR_DT_F32, (in ? p : 0) * D + d0, cs);
  if (!in) {
#pragma unroll
    for (int e = 0; e < 8; ++e) cs[e] = __builtin_nanf("");
  }
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
    r = inv_rms(head_sum<C>(sum_sq(x)), D, a.eps);
  }
  norm_turn(x, a.q_norm == kHead, r, w, a.cs != nullptr, cs);
  if (live) store8(a.q_out, DT, unit * D + d0, x);
}

// A q row with a norm over all of it: a wave per token.
template <int DT, int D>
FVSR_DEV void q_row(const Args& a, int t) {
  if (t >= a.T) return;
  const int lane = threadIdx.x & 63;
  const float r =
      inv_rms(row_sq<DT, D>(a.q, t * a.q_ts, a.q_hs, a.q_heads), a.q_heads * D, a.eps);
  for (int c = lane; c < a.q_heads * (D / 8); c += 64) {
    const int h = c / (D / 8), d0 = (c % (D / 8)) * 8;
    float x[8], w[8], cs[8] = {};
    load8(a.q, DT, t * a.q_ts + h * a.q_hs + d0, x);
    load8(a.q_weight, a.w_dt, c * 8, w);
    if (a.cs) load_turn<D>(a, t, d0, cs);
    norm_turn(x, true, r, w, a.cs != nullptr, cs);
    store8(a.q_out, DT, (int64_t)t * a.q_heads * D + c * 8, x);
  }
}

template <int DT, int D>
FVSR_DEV void q_rows(const Args& a, int64_t wg) {
  if (a.q_norm == kRow)
    q_row<DT, D>(a, (int)(wg * 4 + (threadIdx.x >> 6)));
  else
    q_chunk<DT, D>(a, wg * kThreads + threadIdx.x);
}

// The launch before, for row norms of many tokens: workgroups 0.. the k rows'
// 1/rms, the rest the q rows.
template <int DT, int D>
__global__ __launch_bounds__(kThreads) void kv_rows_kernel(Args a) {
  const int stat_wgs = (a.T + 3) / 4;
  if ((int)blockIdx.x >= stat_wgs) return q_rows<DT, D>(a, blockIdx.x - stat_wgs);
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= a.T) return;
  const int H = (int)a.c.heads;
  const float r = inv_rms(row_sq<DT, D>(a.k, t * a.k_ts, a.k_hs, H), H * D, a.eps);
  if ((threadIdx.x & 63) == 0) a.row_stat[t] = r;
}

// Scale exponent of a largest magnitude, given as its (finite) bits: 448 =
// 1.75 * 2^8, so a mantissa above 1.75 carries into the exponent.
FVSR_DEV int scale_exp(uint32_t top) { return max((int)((top + 0x1fffffu) >> 23) - 135, -126); }

FVSR_DEV uint32_t mag(float x) { return __float_as_uint(x) & 0x7fffffffu; }

FVSR_DEV uint32_t finite_mag(float x) {
  const uint32_t m = mag(x);
  return m < 0x7f800000u ? m : 0u;
}

// Four held codes at another scale: exact but for results below 2^-6.
FVSR_DEV uint32_t rescale4(uint32_t w, float f) {
  typedef float v2f __attribute__((ext_vector_type(2)));
  const v2f a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const v2f b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  return e4m3x4(a[0] * f, a[1] * f, b[0] * f, b[1] * f);
}

FVSR_DEV float pow2(int e) { return __builtin_ldexpf(1.0f, e); }

template <int DT, int D>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(Args a) {
  if ((int)blockIdx.x >= a.page_wgs) return q_rows<DT, D>(a, blockIdx.x - a.page_wgs);
  constexpr int C = D / 8;                  // threads of a token
  constexpr int R = kPage / (kThreads / C);  // tokens of a thread: 8 (D = 128) or 4
  __shared__ uint8_t vt[D * kPage];          // v's codes, [dim][token]
  __shared__ float stat[kPage];
  __shared__ uint32_t tops[4][2];
  const int H = (int)a.c.heads, h = blockIdx.x % H, unit = blockIdx.x / H;
  const int tid = threadIdx.x, wave = tid >> 6;

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
  const int at = s.len - s.rows.n;                  // position of the sequence's first new token
  const int page = max(at, 0) / kPage + s.part;
  if (page >= a.c.table_pages) return;              // past the table: dropped
  const int lo = max(max(at, 0), page * kPage) - page * kPage;
  const int hi = min(s.len - page * kPage, kPage);  // new tokens: slots lo .. hi - 1
  const int64_t id = a.c.table[s.b * a.c.table_stride + page];
  if (id < 0 || id >= a.c.pages) return;            // no such page: dropped
  const int row0 = s.rows.lo + page * kPage - at;   // token of slot 0
  const int64_t ph = id * H + h;
  uint8_t* const ksp = (uint8_t*)a.c.k_scale + ph;
  uint8_t* const vsp = (uint8_t*)a.c.v_scale + ph;
  const int k_old = *ksp - 127, v_old = *vsp - 127;

  // Row norms that no launch before has summed: a wave per token.
  if (a.k_norm == kRow && !a.row_stat) {
    for (int i = lo + wave; i < hi; i += 4) {
      const float r = inv_rms(row_sq<DT, D>(a.k, (row0 + i) * a.k_ts, a.k_hs, H), H * D, a.eps);
      if ((tid & 63) == 0) stat[i] = r;
    }
    __syncthreads();
  }

  const int d0 = (tid % C) * 8, slot0 = tid / C * R;
  float w[8] = {};
  if (a.k_norm == kHead) load8(a.k_weight, a.w_dt, d0, w);
  if (a.k_norm == kRow) load8(a.k_weight, a.w_dt, h * D + d0, w);
  float x[R][8], y[R][8];
  uint32_t kt = 0, vtop = 0;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int slot = slot0 + i;
    const bool live = slot >= lo && slot < hi;
    const int t = row0 + (live ? slot : lo);  // others: a token that exists, as zeros
    float cs[8] = {};
    load8(a.k, DT, t * a.k_ts + h * a.k_hs + d0, x[i]);
    load8(a.v, DT, t * a.v_ts + h * a.v_hs + d0, y[i]);
    if (a.cs) load_turn<D>(a, t, d0, cs);
    float r = 1.0f;
    if (a.k_norm == kHead) r = inv_rms(head_sum<C>(sum_sq(x[i])), D, a.eps);
    if (a.k_norm == kRow) r = a.row_stat ? a.row_stat[t] : stat[t - row0];
    norm_turn(x[i], a.k_norm != kNone, r, w, a.cs != nullptr, cs);
    if (!live) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[i][e] = y[i][e] = 0.0f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      kt = max(kt, finite_mag(x[i][e]));
      vtop = max(vtop, finite_mag(y[i][e]));
    }
  }
  kt = __float_as_uint(wave_max_abs(__uint_as_float(kt)));
  vtop = __float_as_uint(wave_max_abs(__uint_as_float(vtop)));
  if ((tid & 63) == 0) tops[wave][0] = kt, tops[wave][1] = vtop;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) kt = max(kt, tops[i][0]), vtop = max(vtop, tops[i][1]);
  int ke = scale_exp(kt), ve = scale_exp(vtop);
  if (lo > 0) ke = max(ke, k_old), ve = max(ve, v_old);
  if (tid == 0) *ksp = (uint8_t)(ke + 127), *vsp = (uint8_t)(ve + 127);

  uint8_t* const kp = (uint8_t*)a.c.k + ph * kPage * D;
  const float kf = pow2(-ke), vf = pow2(-ve);
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int slot = slot0 + i;
    u32x2_t* const p = (u32x2_t*)(kp + slot * D + d0);
    if (slot >= lo && slot < hi) {
      *p = u32x2_t{e4m3x4(x[i][0] * kf, x[i][1] * kf, x[i][2] * kf, x[i][3] * kf),
                   e4m3x4(x[i][4] * kf, x[i][5] * kf, x[i][6] * kf, x[i][7] * kf)};
    } else if (slot < lo && ke != k_old) {
      const u32x2_t c = *p;
      *p = u32x2_t{rescale4(c[0], pow2(k_old - ke)), rescale4(c[1], pow2(k_old - ke))};
    }
  }
  // [dim][token]: a thread's R tokens of a dim are one unit of R bytes; unit u
  // of row d sits at u ^ (d / 8 % 16), so that the D/8 threads of a token spread
  // over the banks.
  const auto vt_at = [&](int d, int u) { return vt + d * kPage + (u ^ ((d >> 3) & 15)) * R; };
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    uint32_t c[2];
#pragma unroll
    for (int g = 0; g < R / 4; ++g)
      c[g] = e4m3x4(y[4 * g][e] * vf, y[4 * g + 1][e] * vf, y[4 * g + 2][e] * vf,
                    y[4 * g + 3][e] * vf);
    __builtin_memcpy(__builtin_assume_aligned(vt_at(d0 + e, slot0 / R), R), c, R);
  }
  __syncthreads();
  uint8_t* const vp = (uint8_t*)a.c.v + ph * kPage * D;
#pragma unroll
  for (int it = 0; it < D * (kPage / 16) / kThreads; ++it) {
    const int idx = it * kThreads + tid, d = idx / (kPage / 16), s0 = idx % (kPage / 16) * 16;
    const bool grow = s0 < lo && ve != v_old;  // held codes to round again
    if ((s0 + 16 <= lo && !grow) || s0 >= hi) continue;
    u32x4_t c;
#pragma unroll
    for (int g = 0; g < 16 / R; ++g)
      __builtin_memcpy((uint8_t*)&c + g * R,
                       __builtin_assume_aligned(vt_at(d, s0 / R + g), R), R);
    uint8_t* const p = vp + d * kPage + s0;
    if (s0 >= lo && s0 + 16 <= hi) {
      *(u32x4_t*)p = c;
      continue;
    }
    if (grow) {
      u32x4_t o = *(const u32x4_t*)p;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const uint32_t n = rescale4(o[g], pow2(v_old - ve));
        uint32_t m = 0, keep = 0;  // bytes of new tokens; bytes behind them
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int slot = s0 + 4 * g + e;
          if (slot >= hi) keep |= 0xffu << (8 * e);
          else if (slot >= lo) m |= 0xffu << (8 * e);
        }
        o[g] = (c[g] & m) | (o[g] & keep) | (n & ~(m | keep));
      }
      *(u32x4_t*)p = o;
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (s0 + e >= lo && s0 + e < hi) p[e] = (uint8_t)(c[e >> 2] >> (8 * (e & 3)));
    }
  }
}

// Tokens up to which each workgroup sums its own rows for a row norm.
constexpr int64_t kOwnStat = 64;

template <int DT, int D>
void launch(const Args& a, int64_t units, hipStream_t st) {
  Args b = a;
  b.page_wgs = (int)(units * a.c.heads);
  const int64_t q_wgs = !a.q                ? 0
                        : a.q_norm == kRow ? (a.T + 3) / 4
                                           : ((int64_t)a.T * a.q_heads * (D / 8) + kThreads - 1) / kThreads;
  if (a.row_stat) {
    hipLaunchKernelGGL((kv_rows_kernel<DT, D>), dim3((unsigned)((a.T + 3) / 4 + q_wgs)),
                       dim3(kThreads), 0, st, b);
    hipLaunchKernelGGL((kv_append_kernel<DT, D>), dim3((unsigned)b.page_wgs), dim3(kThreads), 0,
                       st, b);
  } else {
    hipLaunchKernelGGL((kv_append_kernel<DT, D>), dim3((unsigned)(b.page_wgs + q_wgs)),
                       dim3(kThreads), 0, st, b);
  }
}

bool rows_aligned(const void* p, int64_t ts, int64_t hs, int64_t size) {
  return (((uintptr_t)p | (uint64_t)(ts * size) | (uint64_t)(hs * size)) & 15) == 0;
}

}  // namespace

extern "C" int64_t fvsr_kv_append_workspace_floats(int64_t T, int k_norm) {
  return k_norm == FVSR_NORM_ROW && T > kOwnStat ? T : 0;
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
  if ((k_norm && !k_weight) || (q && q_norm && !q_weight)) return FVSR_EINVAL;
  if (cs && (cs_rows <= 0 || (!positions && cs_rows < T))) return FVSR_EINVAL;
  if (T == 0 || cache->sequences == 0) return FVSR_OK;
  if (!k || !v) return FVSR_EINVAL;
  const int64_t size = dtype == FVSR_DT_F32 ? 4 : 2, D = cache->head_dim, B = cache->sequences;
  if (!rows_aligned(k, k_tok_stride, k_head_stride, size) ||
      !rows_aligned(v, v_tok_stride, v_head_stride, size) ||
      (q && !rows_aligned(q, q_tok_stride, q_head_stride, size)) ||
      (((uintptr_t)q_out | (uintptr_t)k_weight | (uintptr_t)q_weight | (uintptr_t)cs) & 15))
    return FVSR_EUNSUPPORTED;
  const int64_t need = fvsr_kv_append_workspace_floats(T, k_norm);
  if (need && (!workspace || workspace_floats < need)) return FVSR_EWORKSPACE;
  // Pages that n tokens touch: at most n, and at most (n + 126) / 128 + 1.
  const auto most = [](int64_t n) { return std::min(n, (n + 126) / kPage + 1); };
  Args a{};
  a.c = *cache;
  a.k = k, a.v = v, a.q = q, a.k_weight = k_weight, a.q_weight = q_weight, a.q_out = q_out;
  a.cs = cs, a.positions = positions, a.row_stat = need ? workspace : nullptr;
  a.k_ts = k_tok_stride, a.k_hs = k_head_stride, a.v_ts = v_tok_stride, a.v_hs = v_head_stride;
  a.q_ts = q_tok_stride, a.q_hs = q_head_stride, a.cs_rows = cs_rows;
  a.T = (int)T, a.q_heads = (int)q_heads, a.k_norm = k_norm, a.q_norm = q_norm;
  a.w_dt = weight_dtype, a.eps = eps;
  a.units_max = (int)most(T / B);
  // Packed rows: the sum of those bounds over any B counts that add up to T.
  const int64_t units = cache->cu ? std::min(T, (T + 126 * B) / kPage + B) : B * a.units_max;
  const int64_t q_wgs = q ? (T * q_heads * (D / 8)) / kThreads + T / 4 + 2 : 0;
  if (units * cache->heads + q_wgs > 0x7fffffff || (q && T * q_heads > 0x7fffffff))
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
