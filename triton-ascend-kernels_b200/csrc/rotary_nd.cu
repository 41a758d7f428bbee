// Rotary positions with several axes (time, height, width, ...).
//
// Pair i of the first rot_dim elements of a head, (x_i, x_{i + rot_dim/2}) or
// interleaved (x_2i, x_2i+1), turns by angle_i = positions[t, axis(i)] *
// inv_freq[i]; axis(i) is given by contiguous sections of the pairs.  The
// remaining head_dim - rot_dim elements pass through.  `inverse` turns by
// -angle_i: the transpose of the rotation, i.e. its gradient.
//
// The angle is formed and reduced in 64 bits (as half turns, modulo 2): in
// 32 bits position 1e5 times frequency 1 is already off by 4e-3 radians.
#include "common.cuh"
#include "kernels.h"

namespace tak {

struct RotaryParams {
  const void* x[2]; int64_t sx[2][3];
  void* y[2]; int64_t sy[2][3];
  const int32_t* positions; int64_t sp[2];
  const float* inv_freq;
  int section_end[8];
  int axes, T, H, Hkv, D, rot, interleaved, inverse;
};

__device__ __forceinline__ float2 rotary_cos_sin(const RotaryParams& p, int position, double freq) {
  const double turns = static_cast<double>(position) * freq;  // angle / pi
  const float r = static_cast<float>(turns - 2.0 * rint(0.5 * turns));
  float s, c;
  sincospif(r, &s, &c);
  return make_float2(c, p.inverse ? -s : s);
}

// A CTA walks blocks of TB tokens (and, for few tokens, a share of their heads).
// A block's TB * rot / 2 cosines and sines are made once, while the block before
// it is turned (two tables); each thread then keeps the ones of its piece of a head
// in registers and walks the heads.  VEC = 16 bytes per access where the layout
// allows, else one element.  Bound by the loads in flight: 16381 tokens x 72 heads
// of 128 (fp16) take FIGURE.
template <typename T, int VEC> struct RotVec;
template <typename T> struct RotVec<T, 1> {
  T e[1];
};
template <typename T> struct alignas(16) RotVec<T, 16 / sizeof(T)> {
  uint32_t u[4];
};
// 16-bit types: a word is two elements
template <typename T> __device__ __forceinline__ void rot_interleaved(RotVec<T, 8>& v, const float2* cs) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 e = Elem<T>::unpack2(v.u[k]);
    v.u[k] = Elem<T>::pack2(e.x * cs[k].x - e.y * cs[k].y, e.x * cs[k].y + e.y * cs[k].x);
  }
}
template <typename T> __device__ __forceinline__ void rot_halves(RotVec<T, 8>& a, RotVec<T, 8>& b, const float2* cs) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 e = Elem<T>::unpack2(a.u[k]), f = Elem<T>::unpack2(b.u[k]), c = cs[2 * k], d = cs[2 * k + 1];
    a.u[k] = Elem<T>::pack2(e.x * c.x - f.x * c.y, e.y * d.x - f.y * d.y);
    b.u[k] = Elem<T>::pack2(e.x * c.y + f.x * c.x, e.y * d.y + f.y * d.x);
  }
}
__device__ __forceinline__ void rot_pair(uint32_t& a, uint32_t& b, float2 c) {
  const float e = __uint_as_float(a), f = __uint_as_float(b);
  a = __float_as_uint(e * c.x - f * c.y);
  b = __float_as_uint(e * c.y + f * c.x);
}
template <typename T> __device__ __forceinline__ void rot_interleaved(RotVec<float, 4>& v, const float2* cs) {
  rot_pair(v.u[0], v.u[1], cs[0]);
  rot_pair(v.u[2], v.u[3], cs[1]);
}
template <typename T> __device__ __forceinline__ void rot_halves(RotVec<float, 4>& a, RotVec<float, 4>& b, const float2* cs) {
#pragma unroll
  for (int k = 0; k < 4; ++k) rot_pair(a.u[k], b.u[k], cs[k]);
}
template <typename T> __device__ __forceinline__ void rot_halves(RotVec<T, 1>& a, RotVec<T, 1>& b, const float2* cs) {
  const float e = Elem<T>::to_f(a.e[0]), f = Elem<T>::to_f(b.e[0]);
  a.e[0] = Elem<T>::from_f(e * cs[0].x - f * cs[0].y);
  b.e[0] = Elem<T>::from_f(e * cs[0].y + f * cs[0].x);
}

template <typename T, int VEC, bool IL>
__global__ void __launch_bounds__(256, 4) rotary_nd_kernel(const __grid_constant__ RotaryParams p, int TB, int heads_per_cta) {
  using V = RotVec<T, VEC>;
  extern __shared__ float2 tables[];  // [2][TB][rot / 2]
  const int h0 = blockIdx.y * heads_per_cta, hn = min(heads_per_cta, p.H + p.Hkv - h0);
  const int half = p.rot / 2;
  // items of a head: pieces of VEC pairs (half-split: two vectors; interleaved:
  // VEC / 2 pairs in one vector), then the vectors that pass through
  const int turn = IL && VEC > 1 ? p.rot / VEC : half / VEC, rest = (p.D - p.rot) / VEC, per_head = turn + rest;
  constexpr int NCS = VEC == 1 ? 1 : IL ? VEC / 2 : VEC;  // pairs of a piece
  const int px = per_head < 256 ? per_head : 256, lanes = 256 / px;
  const int hl = threadIdx.x / px;
  const int64_t step = static_cast<int64_t>(gridDim.x) * TB;

  // a thread's table entries have the same pair (and frequency) in every block
  // when TB * half entries fit the threads; else they are looked up each time
  const bool one = TB * half <= 256;
  const int my_t = half > 0 ? threadIdx.x / half : 0, my_i = half > 0 ? threadIdx.x - my_t * half : 0;
  const bool makes = one && my_t < TB && half > 0;
  auto axis_of = [&](int i) {
    int axis = 0;
    while (axis < p.axes - 1 && i >= p.section_end[axis]) ++axis;
    return axis;
  };
  constexpr double kInvPi = 0.31830988618379067154;
  const int axis = makes ? axis_of(my_i) : 0;
  const double freq = makes ? static_cast<double>(p.inv_freq[my_i]) * kInvPi : 0.0;
  auto position = [&](int64_t t0) {
    return makes && t0 + my_t < p.T ? p.positions[(t0 + my_t) * p.sp[0] + axis * p.sp[1]] : 0;
  };
  auto make_table = [&](int64_t t0, int pos, float2* table) {
    if (one) {
      if (makes) table[threadIdx.x] = rotary_cos_sin(p, pos, freq);
    } else {
      for (int e = threadIdx.x; e < TB * half; e += 256) {
        const int ti = e / half, i = e - ti * half;
        if (t0 + ti < p.T)
          table[e] = rotary_cos_sin(p, p.positions[(t0 + ti) * p.sp[0] + axis_of(i) * p.sp[1]],
                                    static_cast<double>(p.inv_freq[i]) * kInvPi);
      }
    }
  };

  int64_t t0 = static_cast<int64_t>(blockIdx.x) * TB;
  int buf = 0;
  make_table(t0, position(t0), tables);
  __syncthreads();
  for (; t0 < p.T; t0 += step, buf ^= 1) {
    const float2* const table = tables + buf * TB * half;
    const int tn = static_cast<int>(min(static_cast<int64_t>(TB), p.T - t0));
    const bool more = t0 + step < p.T;
    const int next_pos = more ? position(t0 + step) : 0;
    for (int ti = 0; ti < tn && hl < lanes; ++ti) {
      const int64_t t = t0 + ti;
      for (int i = threadIdx.x - hl * px; i < per_head; i += px) {
        float2 cs[NCS];
        if (i < turn) {
#pragma unroll
          for (int k = 0; k < NCS; ++k) cs[k] = table[ti * half + i * NCS + k];
        }
        // first element of the piece, and of its partner half
        const int da = i >= turn ? p.rot + (i - turn) * VEC : IL ? (VEC > 1 ? i * VEC : 2 * i) : i * VEC;
        const int db = IL ? da + 1 : da + half;
        // q's heads of this CTA, then k's (apart, so that each has fixed strides)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const int lo = w ? max(h0, p.H) : h0, hi = w ? h0 + hn : min(h0 + hn, p.H), off = w ? p.H : 0;
          const T* const x0 = static_cast<const T*>(p.x[w]) + t * p.sx[w][0];
          T* const y0 = static_cast<T*>(p.y[w]) + t * p.sy[w][0];
          const int64_t dx = VEC > 1 ? 1 : p.sx[w][2], dy = VEC > 1 ? 1 : p.sy[w][2];
          constexpr int MLP = VEC == 1 ? 1 : IL ? 4 : 2;  // heads in flight
          for (int h = lo + hl; h < hi; h += MLP * lanes) {
            V a[MLP], b[MLP];
#pragma unroll
            for (int u = 0; u < MLP; ++u) {
              const int hh = h + u * lanes;
              if (hh < hi) {
                const T* x = x0 + (hh - off) * p.sx[w][1];
                a[u] = *reinterpret_cast<const V*>(x + da * dx);
                if ((!IL || VEC == 1) && i < turn) b[u] = *reinterpret_cast<const V*>(x + db * dx);
              }
            }
#pragma unroll
            for (int u = 0; u < MLP; ++u) {
              const int hh = h + u * lanes;
              if (hh >= hi) continue;
              T* y = y0 + (hh - off) * p.sy[w][1];
              if (i < turn) {
                if constexpr (IL && VEC > 1) {
                  rot_interleaved<T>(a[u], cs);
                } else {
                  rot_halves<T>(a[u], b[u], cs);
                  *reinterpret_cast<V*>(y + db * dy) = b[u];
                }
              }
              *reinterpret_cast<V*>(y + da * dy) = a[u];
            }
          }
        }
      }
    }
    if (more) make_table(t0 + step, next_pos, tables + (buf ^ 1) * TB * half);
    __syncthreads();
  }
}

// 16-byte accesses: unit element strides, rows and base on 16 bytes, and the
// parts of a head (both halves, or the pairs; what passes through) whole vectors.
static bool rotary_vec_ok(const RotaryArgs& a, int vec) {
  const int part = a.interleaved ? a.rot_dim : a.rot_dim / 2;
  if (part % vec || (a.head_dim - a.rot_dim) % vec) return false;
  const int64_t* st[] = {a.sq, a.sqo, a.sk, a.sko};
  const void* base[] = {a.q, a.q_out, a.k, a.k_out};
  for (int i = 0; i < 4; ++i) {
    if ((i < 2 ? a.num_q_heads : a.num_kv_heads) == 0) continue;
    if (st[i][2] != 1 || st[i][0] % vec || st[i][1] % vec || (reinterpret_cast<uintptr_t>(base[i]) & 15)) return false;
  }
  return true;
}

template <typename T>
static void rotary_launch_t(const RotaryArgs& a, const RotaryParams& p, cudaStream_t st) {
  constexpr int VEC = 16 / sizeof(T);
  const bool vec = rotary_vec_ok(a, VEC);
  const int heads = a.num_q_heads + a.num_kv_heads, half = a.rot_dim / 2;
  // tokens of a block: about one table entry a thread; fewer tokens than that fills
  // the GPU with CTAs over shares of the heads instead
  int tb = half > 0 ? 256 / half : 4;
  if (tb > 4) tb = 4;
  if (tb < 1) tb = 1;
  const int want = 4 * num_sms();
  while (tb > 1 && (a.total_tokens + tb - 1) / tb < want) tb = (tb + 1) / 2;
  const int blocks = (a.total_tokens + tb - 1) / tb, ctas = blocks < want ? blocks : want;
  int split = ctas < want / 2 ? want / 2 / ctas : 1;
  if (split > (heads + 3) / 4) split = (heads + 3) / 4;
  const int per = (heads + split - 1) / split;
  const dim3 grid(ctas, (heads + per - 1) / per);
  const size_t smem = static_cast<size_t>(2 * tb) * half * sizeof(float2);
  if (vec && a.interleaved) rotary_nd_kernel<T, VEC, true><<<grid, 256, smem, st>>>(p, tb, per);
  else if (vec) rotary_nd_kernel<T, VEC, false><<<grid, 256, smem, st>>>(p, tb, per);
  else if (a.interleaved) rotary_nd_kernel<T, 1, true><<<grid, 256, smem, st>>>(p, tb, per);
  else rotary_nd_kernel<T, 1, false><<<grid, 256, smem, st>>>(p, tb, per);
}

int rotary_nd_launch(const RotaryArgs& a, cudaStream_t st) {
  RotaryParams p{};
  p.x[0] = a.q; p.x[1] = a.k; p.y[0] = a.q_out; p.y[1] = a.k_out;
  for (int i = 0; i < 3; ++i) {
    p.sx[0][i] = a.sq[i]; p.sx[1][i] = a.sk[i];
    p.sy[0][i] = a.sqo[i]; p.sy[1][i] = a.sko[i];
  }
  p.positions = a.positions; p.sp[0] = a.sp[0]; p.sp[1] = a.sp[1];
  p.inv_freq = a.inv_freq;
  for (int i = 0; i < a.axes; ++i) p.section_end[i] = a.section_end[i];
  p.axes = a.axes; p.T = a.total_tokens; p.H = a.num_q_heads; p.Hkv = a.num_kv_heads;
  p.D = a.head_dim; p.rot = a.rot_dim; p.interleaved = a.interleaved; p.inverse = a.inverse;
  note_kernel("rotary_nd");
  if (a.dtype == kBF16) rotary_launch_t<__nv_bfloat16>(a, p, st);
  else if (a.dtype == kF16) rotary_launch_t<__half>(a, p, st);
  else rotary_launch_t<float>(a, p, st);
  return 0;
}

}  // namespace tak
