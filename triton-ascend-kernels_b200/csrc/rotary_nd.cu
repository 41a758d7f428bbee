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

__device__ __forceinline__ float2 rotary_cos_sin(const RotaryParams& p, int position, float inv_freq) {
  const double turns = static_cast<double>(position) * static_cast<double>(inv_freq) * 0.31830988618379067154;  // angle / pi
  const float r = static_cast<float>(turns - 2.0 * rint(0.5 * turns));
  float s, c;
  sincospif(r, &s, &c);
  return make_float2(c, p.inverse ? -s : s);
}

// A warp turns one token's heads, or a share of them where there are few tokens: it
// makes the token's rot / 2 cosines and sines in shared memory of its own (no CTA
// barrier), each lane keeps the ones of its piece of a head in registers and walks
// the heads, the next heads' loads in flight while it turns these; the first are
// issued before the table is made.  VEC = 16 bytes per access where the layout
// allows, else one element.
//
// Bound by memory: 16381 tokens x 40 heads of 128 (fp16, 96 elements turned) in 57
// us, 5.87 TB/s, 90 % of the measured copy rate.  A CTA per block of four tokens
// with one table behind a CTA barrier took 78 to 84 us, its first loads waiting for
// the table.  One decode step (64 tokens x 40 heads) takes 3.6 us, a launch and two
// memory round trips.
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
__global__ void __launch_bounds__(256, 4) rotary_nd_kernel(const __grid_constant__ RotaryParams p, int shares, int per_share) {
  using V = RotVec<T, VEC>;
  extern __shared__ float2 tables[];  // [8 warps][rot / 2]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int half = p.rot / 2;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 8 + warp;
  const int64_t t = unit / shares;
  if (t >= p.T) return;
  const int h0 = static_cast<int>(unit - t * shares) * per_share, h1 = min(h0 + per_share, p.H + p.Hkv);
  // pieces of a head: VEC pairs (half-split: two vectors; interleaved: VEC / 2 pairs
  // in one vector), then the vectors that pass through
  const int turn = IL && VEC > 1 ? p.rot / VEC : half / VEC, per_head = turn + (p.D - p.rot) / VEC;
  const int px = per_head < 32 ? per_head : 32, lanes = 32 / px, hl = lane / px;
  constexpr int NCS = VEC == 1 ? 1 : IL ? VEC / 2 : VEC;  // pairs of a piece
  constexpr bool TWO = !IL || VEC == 1;                   // a piece is two vectors
  constexpr int MLP = TWO ? 2 : 4;                        // heads in flight
  float2* const table = tables + warp * half;
  bool made = false;

  for (int i0 = 0; i0 < per_head; i0 += px) {
    const int i = i0 + lane - hl * px;
    const bool live = hl < lanes && i < per_head;
    // first element of the piece, and of its partner half
    const int da = i >= turn ? p.rot + (i - turn) * VEC : IL ? (VEC > 1 ? i * VEC : 2 * i) : i * VEC;
    const int db = IL ? da + 1 : da + half;
    float2 cs[NCS];
    // q's heads of this share, then k's (apart, so that each has fixed strides)
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const int lo = (w ? max(h0, p.H) - p.H : h0) + hl, hi = w ? h1 - p.H : min(h1, p.H);
      const int64_t dx = VEC > 1 ? 1 : p.sx[w][2], dy = VEC > 1 ? 1 : p.sy[w][2];
      const T* x = static_cast<const T*>(p.x[w]) + t * p.sx[w][0] + lo * p.sx[w][1] + da * dx;
      T* y = static_cast<T*>(p.y[w]) + t * p.sy[w][0] + lo * p.sy[w][1] + da * dy;
      const int64_t xs = lanes * p.sx[w][1], ys = lanes * p.sy[w][1], xb = (db - da) * dx, yb = (db - da) * dy;
      V a[MLP], b[MLP];
      auto load = [&](int h) {
#pragma unroll
        for (int u = 0; u < MLP; ++u)
          if (live && h + u * lanes < hi) {
            a[u] = *reinterpret_cast<const V*>(x + u * xs);
            if (TWO && i < turn) b[u] = *reinterpret_cast<const V*>(x + u * xs + xb);
          }
        x += MLP * xs;
      };
      load(lo);
      if (!made) {  // the token's table, once, under the first loads
        for (int e = lane; e < half; e += 32) {
          int axis = 0;
          while (axis < p.axes - 1 && e >= p.section_end[axis]) ++axis;
          table[e] = rotary_cos_sin(p, p.positions[t * p.sp[0] + axis * p.sp[1]], p.inv_freq[e]);
        }
        __syncwarp();
        made = true;
      }
      if (w == 0 && live && i < turn) {
#pragma unroll
        for (int k = 0; k < NCS; ++k) cs[k] = table[i * NCS + k];
      }
      for (int h = lo; h < hi; h += MLP * lanes) {
        V c[MLP], d[MLP];
#pragma unroll
        for (int u = 0; u < MLP; ++u) {
          c[u] = a[u];
          if (TWO) d[u] = b[u];
        }
        load(h + MLP * lanes);
#pragma unroll
        for (int u = 0; u < MLP; ++u) {
          if (!live || h + u * lanes >= hi) continue;
          if (i < turn) {
            if constexpr (!TWO) {
              rot_interleaved<T>(c[u], cs);
            } else {
              rot_halves<T>(c[u], d[u], cs);
              *reinterpret_cast<V*>(y + u * ys + yb) = d[u];
            }
          }
          *reinterpret_cast<V*>(y + u * ys) = c[u];
        }
        y += MLP * ys;
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
  // a warp per token; with fewer tokens than warps that fill the GPU, a warp per
  // token and share of its heads (at least four, as each share makes the table)
  int64_t shares = 16 * static_cast<int64_t>(num_sms()) / a.total_tokens;
  if (shares > heads / 4) shares = heads / 4;
  if (shares < 1) shares = 1;
  const int per = (heads + static_cast<int>(shares) - 1) / static_cast<int>(shares);
  shares = (heads + per - 1) / per;
  const unsigned grid = static_cast<unsigned>((a.total_tokens * shares + 7) / 8);
  const size_t smem = static_cast<size_t>(8) * half * sizeof(float2);
  if (vec && a.interleaved) rotary_nd_kernel<T, VEC, true><<<grid, 256, smem, st>>>(p, static_cast<int>(shares), per);
  else if (vec) rotary_nd_kernel<T, VEC, false><<<grid, 256, smem, st>>>(p, static_cast<int>(shares), per);
  else if (a.interleaved) rotary_nd_kernel<T, 1, true><<<grid, 256, smem, st>>>(p, static_cast<int>(shares), per);
  else rotary_nd_kernel<T, 1, false><<<grid, 256, smem, st>>>(p, static_cast<int>(shares), per);
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
