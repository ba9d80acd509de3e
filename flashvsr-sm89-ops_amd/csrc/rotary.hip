// Rotary positions of q and k: the first `turned` channels of each head in pairs,
//
//   (a, b) -> gain * (a cos t - b sin t, a sin t + b cos t),  t = 2 pi frac(position * turns[i])
//
// the pairs (2 i, 2 i + 1) or (i, i + turned / 2); the other channels are copied.  The way
// back (the gradient) has -t.  The product and its fraction are in 64 bits, so an angle of
// position 2^31 is still right to 2^-23 of a turn; sine and cosine are fp32, as is all behind them.
//
// Bound by bytes: each value is read and written once.  A thread has eight pairs of one token
// and turns them in every HS-th head, so that an angle is made once for several heads.
#include <algorithm>

#include "common.h"

namespace {

constexpr int kThreads = 256;

struct Args {
  fvsr_rotary_rows x[2];  // q and k, or q alone (0 heads in the second)
  const double* turns;
  const int32_t* positions;
  int64_t pos_batch, threads;
  int S, D, turned, back;
  int heads, slots, turning, step;  // of both; slots of a head, those that turn; heads' stride
  float gain;
};

template <int DT, int V>
struct Pack {  // V values of type DT as fp32
  float v[V];
};
template <int DT, int V>
FVSR_DEV Pack<DT, V> load(const void* p, int64_t i) {
  Pack<DT, V> r;
  if constexpr (V == 1) {
    r.v[0] = ld_elem(p, DT, i);
  } else if constexpr (DT == FVSR_DT_F32) {
    const f32x4_t a = *(const f32x4_t*)((const float*)p + i), b = *((const f32x4_t*)((const float*)p + i) + 1);
#pragma unroll
    for (int k = 0; k < 4; ++k) r.v[k] = a[k], r.v[4 + k] = b[k];
  } else {
    const u32x4_t w = *(const u32x4_t*)((const uint16_t*)p + i);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t u = w[k];  // (a bit cast of a vector's element would take its first)
      if constexpr (DT == FVSR_DT_F16) {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        const h2 h = __builtin_bit_cast(h2, u);
        r.v[2 * k] = (float)h[0], r.v[2 * k + 1] = (float)h[1];
      } else {
        r.v[2 * k] = bf_lo(u), r.v[2 * k + 1] = bf_hi(u);
      }
    }
  }
  return r;
}
template <int DT, int V>
FVSR_DEV void store(void* p, int64_t i, const Pack<DT, V>& r) {
  if constexpr (V == 1) {
    st_elem(p, DT, i, r.v[0]);
  } else if constexpr (DT == FVSR_DT_F32) {
    f32x4_t* to = (f32x4_t*)((float*)p + i);
    to[0] = f32x4_t{r.v[0], r.v[1], r.v[2], r.v[3]};
    to[1] = f32x4_t{r.v[4], r.v[5], r.v[6], r.v[7]};
  } else {
    u32x4_t w;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (DT == FVSR_DT_F16) {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        w[k] = __builtin_bit_cast(uint32_t, h2{(_Float16)r.v[2 * k], (_Float16)r.v[2 * k + 1]});
      } else {
        w[k] = pack_bf16x2(r.v[2 * k], r.v[2 * k + 1]);
      }
    }
    *(u32x4_t*)((uint16_t*)p + i) = w;
  }
}

template <int DT, int V, bool HALF>
__global__ __launch_bounds__(kThreads) void rotary_kernel(Args a) {
  const int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (at >= a.threads) return;
  const int slot = (int)(at % a.slots);
  const int64_t group = at / a.slots;
  const int h0 = (int)(group % a.step);
  const int64_t row = group / a.step, b = row / a.S;
  const int s = (int)(row % a.S);
  const bool turns = slot < a.turning;
  // Channels of the slot: V pairs, or 2 V that are copied (the last slot may have V).
  const int c0 = !turns ? a.turned + (slot - a.turning) * 2 * V : HALF ? slot * V : slot * 2 * V;
  const int c1 = turns && HALF ? c0 + a.turned / 2 : c0 + V;
  const bool both = c1 < a.D;
  float cs[V], sn[V];
  if (turns) {
    const double pos = a.positions ? a.positions[b * a.pos_batch + s] : s;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      double t = pos * a.turns[slot * V + i];
      t -= __builtin_rint(t);
      float y, x;
      sincospif((float)(t + t), &y, &x);
      cs[i] = x * a.gain, sn[i] = (a.back ? -y : y) * a.gain;
    }
  }
  for (int h = h0; h < a.heads; h += a.step) {
    const bool k = h >= a.x[0].heads;
    const fvsr_rotary_rows& x = a.x[k];
    const int64_t hh = h - (k ? a.x[0].heads : 0);
    const int64_t from = b * x.x_batch + s * x.x_tok + hh * x.x_head;
    const int64_t to = (row * x.heads + hh) * a.D;
    Pack<DT, V> p = load<DT, V>(x.x, from + c0), q = p;
    if (both) q = load<DT, V>(x.x, from + c1);
    if (turns) {
      // Pairs (p[i], q[i]), or neighbours in p, then in q.
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float& u = HALF || V == 1 ? p.v[i] : i < V / 2 ? p.v[2 * i] : q.v[2 * i - V];
        float& v = HALF || V == 1 ? q.v[i] : i < V / 2 ? p.v[2 * i + 1] : q.v[2 * i + 1 - V];
        const float u0 = u;
        u = u0 * cs[i] - v * sn[i];
        v = u0 * sn[i] + v * cs[i];
      }
    }
    store<DT, V>(x.y, to + c0, p);
    if (both) store<DT, V>(x.y, to + c1, q);
  }
}

template <int DT, int V>
void launch(const Args& a, bool half, hipStream_t st) {
  const dim3 grid((unsigned)((a.threads + kThreads - 1) / kThreads));
  if (half)
    hipLaunchKernelGGL((rotary_kernel<DT, V, true>), grid, dim3(kThreads), 0, st, a);
  else
    hipLaunchKernelGGL((rotary_kernel<DT, V, false>), grid, dim3(kThreads), 0, st, a);
}
template <int DT>
void launch(const Args& a, bool vec, bool half, hipStream_t st) {
  vec ? launch<DT, 8>(a, half, st) : launch<DT, 1>(a, half, st);
}

}  // namespace

extern "C" int fvsr_rotary(const fvsr_rotary_rows* q, const fvsr_rotary_rows* k, int dtype,
                           int64_t batch, int64_t tokens, int64_t head_dim, int64_t turned,
                           const double* turns, const int32_t* positions, int64_t pos_batch_stride,
                           float gain, int pairs, int back, void* stream) {
  if (!q || batch < 0 || tokens < 0 || head_dim <= 0 || turned < 0 || turned > head_dim ||
      turned % 2 || (pairs != FVSR_PAIRS_HALF && pairs != FVSR_PAIRS_INTERLEAVED))
    return FVSR_EINVAL;
  if (dtype != FVSR_DT_BF16 && dtype != FVSR_DT_F16 && dtype != FVSR_DT_F32) return FVSR_EINVAL;
  if (head_dim > (1 << 20) || tokens > 0x7fffffff || batch > 0x7fffffff) return FVSR_EUNSUPPORTED;
  Args a{};
  a.x[0] = *q;
  if (k) a.x[1] = *k;
  const int64_t rows = batch * tokens, size = dtype == FVSR_DT_F32 ? 4 : 2;
  bool vec = turned % 16 == 0 && head_dim % 8 == 0;
  for (const fvsr_rotary_rows& x : a.x) {
    if (x.heads < 0 || x.heads > (1 << 24)) return FVSR_EINVAL;
    if (x.heads == 0 || rows == 0) continue;
    if (!x.x || !x.y) return FVSR_EINVAL;
    if (((uintptr_t)x.x | (uintptr_t)x.y) & (size - 1)) return FVSR_EUNSUPPORTED;
    vec = vec && !(((uintptr_t)x.x | (uintptr_t)x.y | (uint64_t)(x.x_batch * size) |
                    (uint64_t)(x.x_tok * size) | (uint64_t)(x.x_head * size)) & 15);
  }
  a.heads = (int)(a.x[0].heads + a.x[1].heads);
  if (rows == 0 || a.heads == 0) return FVSR_OK;
  if (turned && (!turns || ((uintptr_t)turns & 7))) return FVSR_EINVAL;
  const int V = vec ? 8 : 1;
  a.turns = turns, a.positions = positions, a.pos_batch = pos_batch_stride;
  a.S = (int)tokens, a.D = (int)head_dim, a.turned = (int)turned, a.back = back != 0;
  a.turning = (int)(turned / 2 / V);
  a.slots = a.turning + (int)((head_dim - turned + 2 * V - 1) / (2 * V));
  a.gain = gain;
  a.step = a.heads;
  if (rows > ((int64_t)1 << 40) / a.slots / a.heads) return FVSR_EUNSUPPORTED;
  a.threads = rows * a.slots * a.step;
  if (a.threads > kThreads * (int64_t)0xffffff) return FVSR_EUNSUPPORTED;
  const hipStream_t st = (hipStream_t)stream;
  const bool half = pairs == FVSR_PAIRS_HALF;
  if (dtype == FVSR_DT_F32)
    launch<FVSR_DT_F32>(a, vec, half, st);
  else if (dtype == FVSR_DT_F16)
    launch<FVSR_DT_F16>(a, vec, half, st);
  else
    launch<FVSR_DT_BF16>(a, vec, half, st);
  return fvsr_launch_status();
}
