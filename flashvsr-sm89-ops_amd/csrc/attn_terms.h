// What the attention kernels over an 8-bit paged cache share (paged_attn.hip,
// selected_attn.hip): operands as sums of e4m3 terms, the softmax's weights at the
// scale of the keys at hand, NaN codes under a mask, and the joining of pieces.  Why the
// operands are split and what precision that leaves stands in paged_attn.hip.
#pragma once
#include "kv_pages.h"

namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v2s __attribute__((ext_vector_type(2)));
#define LDS_AS __attribute__((address_space(3)))

constexpr int kThreads = 256;
constexpr float kNothing = -1e30f;  // reference of a row that has seen no key (finite)
constexpr int kMaxSplits = 64;
constexpr int64_t kMaxGridYZ = 65535;

template <int DT>
FVSR_DEV float to_f(uint16_t x) {
  return DT == FVSR_DT_F16 ? (float)__builtin_bit_cast(_Float16, x) : bf2f(x);
}
template <int DT>
FVSR_DEV uint32_t pack2(float a, float b) {
  if (DT == FVSR_DT_F16) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, h2{(_Float16)a, (_Float16)b});
  }
  return pack_bf16x2(a, b);
}

constexpr int terms(int dt) { return dt == FVSR_DT_F16 ? 3 : 2; }

// Four values of magnitude at most 256 as N e4m3 terms: x = t0 + t1 / 32 + t2 / 1024.
template <int N>
FVSR_DEV void split4(float a, float b, float c, float d, uint32_t (&w)[N]) {
  const uint32_t t0 = e4m3x4(a, b, c, d);
  w[0] = t0;
  if constexpr (N > 1) {
    const v2f lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)t0, false);
    const v2f hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)t0, true);
    a -= lo[0], b -= lo[1], c -= hi[0], d -= hi[1];
    // (Both halves of a destination are written; what it held does not matter.)
    v2s t = __builtin_bit_cast(v2s, a);
    t = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(t, a, b, 0x1p-5f, false);
    t = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(t, c, d, 0x1p-5f, true);
    w[1] = __builtin_bit_cast(uint32_t, t);
  }
  if constexpr (N > 2) {
    const v2f lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[1], 0x1p-5f, false);
    const v2f hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[1], 0x1p-5f, true);
    v2s t = __builtin_bit_cast(v2s, a);
    t = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(t, a - lo[0], b - lo[1], 0x1p-10f, false);
    t = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(t, c - hi[0], d - hi[1], 0x1p-10f, true);
    w[2] = __builtin_bit_cast(uint32_t, t);
  }
}

// Four weights (0 to 256) as N e4m3 terms; `sum` grows by them.  Two terms (8
// bits) come by way of fp16 (11 bits), whose pairs convert, subtract and sum two at a
// time: 24 instructions for 8 weights against 32.  The sum is of the same fp16 values.
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
template <int N>
FVSR_DEV void weights4(float a, float b, float c, float d, uint32_t (&w)[N], float& sum) {
  if constexpr (N == 2) {
    v2h x = {(_Float16)a, (_Float16)b}, y = {(_Float16)c, (_Float16)d};
    const v2h one = {(_Float16)1.0f, (_Float16)1.0f};
    sum = __builtin_amdgcn_fdot2(x, one, sum, false);
    sum = __builtin_amdgcn_fdot2(y, one, sum, false);
    // (Both halves of a destination are written; what it held does not matter.)
    v2s o = __builtin_bit_cast(v2s, x);
    o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(o, x, 1.0f, false);
    o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(o, y, 1.0f, true);
    w[0] = __builtin_bit_cast(uint32_t, o);
    x -= __builtin_bit_cast(v2h, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[0], 1.0f, false));
    y -= __builtin_bit_cast(v2h, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[0], 1.0f, true));
    o = __builtin_bit_cast(v2s, x);
    o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(o, x, 0x1p-5f, false);
    o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(o, y, 0x1p-5f, true);
    w[1] = __builtin_bit_cast(uint32_t, o);
  } else {
    sum += (a + b) + (c + d);
    split4<N>(a, b, c, d, w);
  }
}

FVSR_DEV int e8m0(int e) { return min(max(e + 127, 0), 254); }

// Exponent e with the row's largest magnitude in [2^7, 2^8) * 2^e.  A row
// with an infinity or NaN keeps it in its codes: all its logits are NaN.
FVSR_DEV int row_exp(uint32_t top) { return max((int)(top >> 23) - 127, -100) - 7; }

FVSR_DEV uint32_t max_mag(uint32_t m, float x) { return max(m, __float_as_uint(x) & 0x7fffffffu); }

// Whether any of a V operand's codes is NaN (0x7f with either sign).
FVSR_DEV bool has_nan(const v8i& v) {
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) any |= ((uint32_t)v[i] & 0x7f7f7f7fu) + 0x01010101u;
  return (any & 0x80808080u) != 0;
}
// Bytes 0x38 (1.0) where a code is NaN; `v` loses them.
FVSR_DEV v8i take_nan(v8i& v) {
  v8i ones;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t hit = (((uint32_t)v[i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
    const uint32_t mask = (hit >> 7) * 0xffu;
    ones[i] = (int)(mask & 0x38383838u);
    v[i] = (int)((uint32_t)v[i] & ~mask);
  }
  return ones;
}

FVSR_DEV v4f mfma(const v8i& a, const v8i& b, const v4f& c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, sa, 0, sb);
}
FVSR_DEV v16f mfma(const v8i& a, const v8i& b, const v16f& c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, sa, 0, sb);
}

FVSR_DEV v8i join(u32x4_t a, u32x4_t b) {
  return v8i{(int)a[0], (int)a[1], (int)a[2], (int)a[3],
             (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
}

// The softmax of one row's N logits at hand (in s; -inf: hidden): s becomes
// the weights, E - 8 - M goes to `shift`, and the reference M moves if need be
// (`rescale` then multiplies O).  Every lane of a row calls it with the row's largest
// logit; the sum of the weights, times 2^shift, is still to be added to l.  `hide`, if given, is
// added to every exponent: -inf where a row sees none of finite logits (top then -inf), else 0.
template <class Acc, int N, class Rescale, class... Hide>
FVSR_DEV void weigh(Acc (&s)[N], float top, float c, float& m, float& l, int& shift,
                    Rescale rescale, Hide... hide) {
  constexpr int E = sizeof(Acc) / 4;
  const float e = fmaxf(__builtin_ceilf(top * c), kNothing);
  if (__ballot(e > m + 64.0f) != 0) {
    asm volatile("" :::);  // a branch: rare after a row's first keys
    const float to = e > m + 64.0f ? e : m;
    const float f = __builtin_amdgcn_exp2f(m - to);
    m = to;
    l *= f;
    rescale(f);
  }
  const float off = ((8.0f - e) + ... + hide);
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < E; ++j)
      s[i][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][j], c, off));
  shift = (int)fmaxf(e - m, -300.0f) - 8;
}

FVSR_DEV int range_at(int pages, int s, int splits) { return (int)((int64_t)pages * s / splits); }

// Workgroups go round robin over the 8 XCDs; each XCD takes a contiguous range of
// `total` units, whose neighbours read the same pages.
FVSR_DEV int xcd_order(int wg, int total) {
  const int per = total / 8, rem = total % 8, xcd = wg % 8, loc = wg / 8;
  return xcd < rem ? xcd * (per + 1) + loc : rem * (per + 1) + (xcd - rem) * per + loc;
}

// A workgroup adds the n pieces of a row: O at o + k * o_step, (M, l) at ml + k *
// ml_step; 4 dims a thread, 8 or 16 pieces at once.
template <int DT, int D>
FVSR_DEV void join_row(const float* po, int64_t o_step, const float* ml, int64_t ml_step, int n,
                       uint16_t* out) {
  constexpr int L = D / 4, G = kThreads / L;
  __shared__ __attribute__((aligned(16))) float part[kThreads / 64][D];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = threadIdx.x / L;
  const float m = lane < n ? ml[lane * ml_step] : kNothing;
  const float l = lane < n ? ml[lane * ml_step + 1] : 0.0f;
  const float f = __builtin_amdgcn_exp2f(m - wave_max(m));
  const float sum = wave_sum(f * l);
  v4f o = {};
  // (Every lane takes every turn: a lane that has left could not lend its factor.)
  for (int s0 = 0; s0 < n; s0 += G) {
    const int s = s0 + group;
    const float w = __shfl(f, s & 63);
    if (s < n) o += *(const v4f*)(po + s * o_step + (lane % L) * 4) * w;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int d = L; d < 64; d *= 2) o[e] += __shfl_xor(o[e], d);
  if (lane < L) *(v4f*)&part[wave][lane * 4] = o;
  __syncthreads();
  if (threadIdx.x >= L) return;
#pragma unroll
  for (int w = 1; w < kThreads / 64; ++w) o += *(const v4f*)&part[w][lane * 4];
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  *(u32x2_t*)(out + lane * 4) =
      u32x2_t{pack2<DT>(o[0] * inv, o[1] * inv), pack2<DT>(o[2] * inv, o[3] * inv)};
}

// Compute units of the current device, a multiple of the 8 XCDs.
int64_t cu_count() {
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess ||
      cus < 8)
    cus = 256;
  return cus & ~7;
}

}  // namespace
