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

__device__ __forceinline__ float2 rotary_cos_sin(const RotaryParams& p, int t, int i) {
  int axis = 0;
  while (axis < p.axes - 1 && i >= p.section_end[axis]) ++axis;
  const double turns = static_cast<double>(p.positions[t * p.sp[0] + axis * p.sp[1]]) *
                       static_cast<double>(p.inv_freq[i]) * 0.31830988618379067154;  // angle / pi
  const float r = static_cast<float>(turns - 2.0 * rint(0.5 * turns));
  float s, c;
  sincospif(r, &s, &c);
  return make_float2(c, p.inverse ? -s : s);
}

// A CTA turns TB tokens (and, for few tokens, a share of their heads): the table
// of TB * rot / 2 cosines and sines is made once; each thread then keeps the ones
// of its piece of a head in registers and walks the heads.  VEC = 16 bytes per
// access where the layout allows, else one element.
template <typename T, int VEC> struct RotVec;
template <typename T> struct RotVec<T, 1> {
  T e[1];
};
template <typename T> struct alignas(16) RotVec<T, 16 / sizeof(T)> {
  T e[16 / sizeof(T)];
};

template <typename T, int VEC, bool IL>
__global__ void __launch_bounds__(256, 4) rotary_nd_kernel(const __grid_constant__ RotaryParams p, int TB, int heads_per_cta) {
  using V = RotVec<T, VEC>;
  extern __shared__ float2 table[];  // [TB][rot / 2]
  const int t0 = blockIdx.x * TB, tn = min(TB, p.T - t0);
  const int h0 = blockIdx.y * heads_per_cta, hn = min(heads_per_cta, p.H + p.Hkv - h0);
  const int half = p.rot / 2;
  // items of a head: pieces of VEC pairs (half-split: two vectors; interleaved:
  // VEC / 2 pairs in one vector), then the vectors that pass through
  const int turn = IL && VEC > 1 ? p.rot / VEC : half / VEC, rest = (p.D - p.rot) / VEC, per_head = turn + rest;
  for (int i = threadIdx.x; i < tn * half; i += 256) table[i] = rotary_cos_sin(p, t0 + i / half, i % half);
  __syncthreads();
  constexpr int NCS = VEC == 1 ? 1 : IL ? VEC / 2 : VEC;  // pairs of a piece
  const int px = per_head < 256 ? per_head : 256, lanes = 256 / px;
  const int hl = threadIdx.x / px;
  if (hl >= lanes) return;
  for (int ti = 0; ti < tn; ++ti) {
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
              if (IL && VEC > 1) {
#pragma unroll
                for (int k = 0; k < VEC / 2; ++k) {
                  const float e = Elem<T>::to_f(a[u].e[(2 * k) % VEC]), f = Elem<T>::to_f(a[u].e[(2 * k + 1) % VEC]);
                  a[u].e[(2 * k) % VEC] = Elem<T>::from_f(e * cs[k % NCS].x - f * cs[k % NCS].y);
                  a[u].e[(2 * k + 1) % VEC] = Elem<T>::from_f(e * cs[k % NCS].y + f * cs[k % NCS].x);
                }
              } else {
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                  const float e = Elem<T>::to_f(a[u].e[k]), f = Elem<T>::to_f(b[u].e[k]);
                  a[u].e[k] = Elem<T>::from_f(e * cs[k % NCS].x - f * cs[k % NCS].y);
                  b[u].e[k] = Elem<T>::from_f(e * cs[k % NCS].y + f * cs[k % NCS].x);
                }
                *reinterpret_cast<V*>(y + db * dy) = b[u];
              }
            }
            *reinterpret_cast<V*>(y + da * dy) = a[u];
          }
        }
      }
    }
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
  // tokens of a CTA: about one table entry a thread; fewer tokens than that fills
  // the GPU with CTAs over shares of the heads instead
  int tb = half > 0 ? (256 + half - 1) / half : 4;
  if (tb > 4) tb = 4;
  const int want = 2 * num_sms();
  while (tb > 1 && (a.total_tokens + tb - 1) / tb < want) tb = (tb + 1) / 2;
  const int blocks = (a.total_tokens + tb - 1) / tb;
  int split = blocks < want ? (want + blocks - 1) / blocks : 1;
  if (split > (heads + 3) / 4) split = (heads + 3) / 4;
  const int per = (heads + split - 1) / split;
  const dim3 grid(blocks, (heads + per - 1) / per);
  const size_t smem = static_cast<size_t>(tb) * half * sizeof(float2);
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
