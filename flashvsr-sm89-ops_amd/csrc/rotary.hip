// Rotary positions of q and k: the first `turned` channels of each head in pairs,
//
//   (a, b) -> gain * (a cos t - b sin t, a sin t + b cos t),  t = 2 pi frac(position * turns[i])
//
// the pairs (2 i, 2 i + 1) or (i, i + turned / 2); the other channels are copied.  The way
// back (the gradient) has -t.  The product and its fraction are in 64 bits, so an angle of
// position 2^31 is still right to 2^-23 of a turn; sine and cosine are fp32, as is all behind them.
// The angle they are of is fp32 too: for fp32 results what its rounding leaves, d, is made up for by
// cos(t + d) = cos t - d sin t and sin(t + d) = sin t + d cos t (d^2 < 2^-46).
//
// Bound by bytes: each value is read and written once.  A thread has two 16-byte pieces of one
// token, at the same place in both halves of the channels that turn, which is whole pairs in either
// layout and lets lanes read whole lines.  It turns them in every apart-th head, so that an angle is
// made once for several heads, with the loads of four heads on their way together.
//
// Measured: 16384 rows x 32 + 8 heads of 128 in bf16 72 us (4.6 TB/s; a copy reaches 5.2), a head
// to a thread 89; 16896 x 24 heads of 128, 64 channels turned, fp32 87 us (4.75 TB/s), with interleaved
// pieces beside one another 104.
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
  int slots, turning, apart;  // slots of a head, those that turn; distance of a thread's heads
  float gain;
};

// V channels of a type as fp32: 16 bytes of them, or one.
template <int V>
struct Pack {
  float v[V];
};
template <int DT, int V>
FVSR_DEV Pack<V> load(const void* p, int64_t i) {
  Pack<V> r;
  if constexpr (V == 1) {
    r.v[0] = ld_elem(p, DT, i);
  } else if constexpr (DT == FVSR_DT_F32) {
    const f32x4_t w = *(const f32x4_t*)((const float*)p + i);
#pragma unroll
    for (int k = 0; k < 4; ++k) r.v[k] = w[k];
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
FVSR_DEV void store(void* p, int64_t i, const Pack<V>& r) {
  if constexpr (V == 1) {
    st_elem(p, DT, i, r.v[0]);
  } else if constexpr (DT == FVSR_DT_F32) {
    *(f32x4_t*)((float*)p + i) = f32x4_t{r.v[0], r.v[1], r.v[2], r.v[3]};
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
  constexpr int U = 4;
  const int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (at >= a.threads) return;
  // Slots of a head stand beside one another, then heads, then tokens.
  const uint32_t each = (uint32_t)(a.slots * a.apart);
  const int64_t row = at <= 0xffffffff ? (uint32_t)at / each : at / each;
  const uint32_t rest = (uint32_t)(at - row * each);
  const int h0 = (int)(rest / (uint32_t)a.slots), slot = (int)(rest % (uint32_t)a.slots);
  const int64_t b = row <= 0x7fffffff ? (uint32_t)row / (uint32_t)a.S : row / a.S;
  const int s = (int)(row - b * a.S);
  const bool turns = slot < a.turning;
  // The slot's two pieces.  (One channel each: interleaved neighbours.)
  const bool side = V == 1 && !HALF;
  const int part = turns ? slot : slot - a.turning, base = turns ? 0 : a.turned;
  const int c0 = turns && side ? 2 * slot : base + part * V;
  const int c1 = turns && side ? c0 + 1 : c0 + (turns ? a.turning : a.slots - a.turning) * V;
  const bool both = c1 < a.D;
  float cs[V], sn[V];
#pragma unroll
  for (int i = 0; i < V; ++i) cs[i] = 1.0f, sn[i] = 0.0f;
  if (turns) {
    const double pos = a.positions ? a.positions[b * a.pos_batch + s] : s;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      // Pair i of the slot: (p[i], q[i]), or neighbours in p, then in q.
      const int pair = HALF || V == 1 ? slot * V + i
                                      : slot * (V / 2) + i % (V / 2) +
                                            (i < V / 2 ? 0 : a.turning * (V / 2));
      double t = pos * a.turns[pair];
      t -= __builtin_rint(t);
      float y, x;
      sincospif((float)(t + t), &y, &x);
      if constexpr (DT == FVSR_DT_F32) {
        const float d = (float)(t + t - (float)(t + t)) * 3.14159265f, x0 = x;
        x -= d * y, y += d * x0;
      }
      cs[i] = x * a.gain, sn[i] = (a.back ? -y : y) * a.gain;
    }
  }
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const fvsr_rotary_rows& x = a.x[n];
    const int heads = (int)x.heads;
    const int64_t from = b * x.x_batch + s * x.x_tok, to = row * heads * a.D;
    for (int h1 = h0; h1 < heads; h1 += U * a.apart) {
      Pack<V> p[U], q[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = h1 + u * a.apart;
        if (h >= heads) continue;
        p[u] = load<DT, V>(x.x, from + h * x.x_head + c0);
        q[u] = p[u];
        if (both) q[u] = load<DT, V>(x.x, from + h * x.x_head + c1);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = h1 + u * a.apart;
        if (h >= heads) continue;
        if (turns) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            float& f = HALF || V == 1 ? p[u].v[i] : i < V / 2 ? p[u].v[2 * i] : q[u].v[2 * i - V];
            float& g = HALF || V == 1 ? q[u].v[i]
                       : i < V / 2    ? p[u].v[2 * i + 1]
                                      : q[u].v[2 * i + 1 - V];
            const float f0 = f;
            f = f0 * cs[i] - g * sn[i];
            g = f0 * sn[i] + g * cs[i];
          }
        }
        store<DT, V>(x.y, to + (int64_t)h * a.D + c0, p[u]);
        if (both) store<DT, V>(x.y, to + (int64_t)h * a.D + c1, q[u]);
      }
    }
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
  vec ? launch<DT, DT == FVSR_DT_F32 ? 4 : 8>(a, half, st) : launch<DT, 1>(a, half, st);
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
  bool vec = turned % (32 / size) == 0 && head_dim % (16 / size) == 0;
  for (const fvsr_rotary_rows& x : a.x) {
    if (x.heads < 0 || x.heads > (1 << 24)) return FVSR_EINVAL;
    if (x.heads == 0 || rows == 0) continue;
    if (!x.x || !x.y) return FVSR_EINVAL;
    if (((uintptr_t)x.x | (uintptr_t)x.y) & (size - 1)) return FVSR_EUNSUPPORTED;
    vec = vec && !(((uintptr_t)x.x | (uintptr_t)x.y | (uint64_t)(x.x_batch * size) |
                    (uint64_t)(x.x_tok * size) | (uint64_t)(x.x_head * size)) & 15);
  }
  const int64_t heads = std::max(a.x[0].heads, a.x[1].heads);
  if (rows == 0 || heads == 0) return FVSR_OK;
  if (turned && (!turns || ((uintptr_t)turns & 7))) return FVSR_EINVAL;
  const int V = vec ? (int)(16 / size) : 1;
  a.turns = turns, a.positions = positions, a.pos_batch = pos_batch_stride;
  a.S = (int)tokens, a.D = (int)head_dim, a.turned = (int)turned, a.back = back != 0;
  a.turning = (int)(turned / 2 / V);
  a.slots = a.turning + (int)((head_dim - turned + 2 * V - 1) / (2 * V));
  a.gain = gain;
  if (rows > ((int64_t)1 << 40) / a.slots / heads) return FVSR_EUNSUPPORTED;
  // Heads of a thread: as many as leave 2^19 threads, two thirds of what the CUs hold, at most 8.
  const int64_t of = std::min<int64_t>(8, std::max<int64_t>(1, rows * a.slots * heads >> 19));
  a.apart = (int)((heads + of - 1) / of);
  a.threads = rows * a.slots * a.apart;
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
