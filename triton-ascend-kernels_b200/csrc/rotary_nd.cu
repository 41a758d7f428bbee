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

template <typename T>
__global__ void __launch_bounds__(256) rotary_nd_kernel(const RotaryParams p) {
  extern __shared__ float2 table[];  // [rot / 2]
  const int t = blockIdx.x, half = p.rot / 2, rest = p.D - p.rot;
  for (int i = threadIdx.x; i < half; i += blockDim.x) table[i] = rotary_cos_sin(p, t, i);
  __syncthreads();
  const int per_head = half + rest;
  const int n = (p.H + p.Hkv) * per_head;
  for (int e = threadIdx.x; e < n; e += blockDim.x) {
    int h = e / per_head;
    const int i = e - h * per_head;
    const int w = h >= p.H;
    if (w) h -= p.H;
    const T* x = static_cast<const T*>(p.x[w]) + t * p.sx[w][0] + h * p.sx[w][1];
    T* y = static_cast<T*>(p.y[w]) + t * p.sy[w][0] + h * p.sy[w][1];
    const int64_t dx = p.sx[w][2], dy = p.sy[w][2];
    if (i < half) {
      const int a = p.interleaved ? 2 * i : i, b = p.interleaved ? 2 * i + 1 : i + half;
      const float u = Elem<T>::to_f(x[a * dx]), v = Elem<T>::to_f(x[b * dx]);
      const float2 cs = table[i];
      y[a * dy] = Elem<T>::from_f(u * cs.x - v * cs.y);
      y[b * dy] = Elem<T>::from_f(u * cs.y + v * cs.x);
    } else {
      const int d = p.rot + i - half;
      y[d * dy] = x[d * dx];
    }
  }
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
  const size_t smem = static_cast<size_t>(a.rot_dim / 2) * sizeof(float2);
  note_kernel("rotary_nd");
  if (a.dtype == kBF16) rotary_nd_kernel<__nv_bfloat16><<<a.total_tokens, 256, smem, st>>>(p);
  else if (a.dtype == kF16) rotary_nd_kernel<__half><<<a.total_tokens, 256, smem, st>>>(p);
  else rotary_nd_kernel<float><<<a.total_tokens, 256, smem, st>>>(p);
  return 0;
}

}  // namespace tak
