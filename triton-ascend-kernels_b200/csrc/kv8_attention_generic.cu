// Attention over the 8-bit KV cache on CUDA cores: any element type (fp32
// too), strides, head dims up to 640, page and group sizes.  One CTA of 4
// warps per query row and head; each warp walks every fourth key with the
// lanes across the head dim, then the warps merge.  Attention weights come
// from a second launch, one warp per key, that recomputes the scores against
// the finished log-sum-exp.  Bound by issue slots and the row's chain of shuffles and
// exponentials; every query row reads the cache again (64 x <= 8192 keys, 32 heads of
// 128, bf16: 11.0 ms against 0.1 on tensor cores), so it serves the shapes that those
// do not take.
//
// The values are summed against a reference of their own: with vs = 2^E v, 1/2 <= v
// < 1, acc = sum_j 2^((s_j - rs) + (E_j - re)) v_j Vc_j, (rs, re) the score and the
// exponent of the key with the largest s_j + E_j.  So a weight too small for fp32
// under a large V keeps its part, and sums of values near fp32's largest stay finite.
#include "kv8.cuh"

namespace tak {

struct Kv8GenericParams {
  Kv8View c;
  const void* q; int64_t sq[4];
  const int32_t* context_lens;
  void* out; int64_t so[4];
  float* lse;   // [B, Lq, H], may be null
  float* lse2;  // [B, Lq, H] base-2 log-sum-exp for the weights pass, may be null
  float* weights; int64_t sw[3];
  int64_t width;
  int H, Lq, G;
  float scale, softcap;
};

constexpr int kKv8MaxPerLane = 20;  // head_dim <= 640

// score in base-2 units
__device__ __forceinline__ float kv8_score2(float dot, float scale, float softcap) {
  const float z = dot * scale;
  if (softcap > 0.f) return softcap * tanhf(z / softcap) * kLog2e;
  return z * kLog2e;
}

template <typename T, int CODE>
__global__ void __launch_bounds__(128) kv8_attention_generic_kernel(const Kv8GenericParams p) {
  const Kv8View& c = p.c;
  const int h = blockIdx.x, i = blockIdx.y, s = blockIdx.z, kvh = h / p.G;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t ctx = min(static_cast<int64_t>(p.context_lens[s]), c.max_rows);
  const int64_t lim = ctx - p.Lq + i + 1;  // keys that this row sees
  const T* q = static_cast<const T*>(p.q) + s * p.sq[0] + i * p.sq[1] + h * p.sq[2];
  float qr[kKv8MaxPerLane], acc[kKv8MaxPerLane];
#pragma unroll
  for (int e = 0; e < kKv8MaxPerLane; ++e) {
    const int d = lane + 32 * e;
    qr[e] = d < c.D ? Elem<T>::to_f(q[d * p.sq[3]]) : 0.f;
    acc[e] = 0.f;
  }
  float m = -INFINITY, l = 0.f, rs = -INFINITY;
  int re = 0;
  for (int64_t r = warp; r < lim; r += 4) {
    const int64_t page = kv8_page(c, s, r);
    const int row = static_cast<int>(r % c.P);
    float dot = 0.f, vs = 0.f;
    const uint8_t* vr = nullptr;
    if (page >= 0) {
      const uint8_t* kr = kv8_row(c.plane[0], page, kvh, row);
      vr = kv8_row(c.plane[1], page, kvh, row);
      vs = *kv8_scale(c.plane[1], page, kvh, row / c.group);
#pragma unroll
      for (int e = 0; e < kKv8MaxPerLane; ++e) {
        const int d = lane + 32 * e;
        if (d < c.D) dot += qr[e] * Kv8<CODE>::dec(kr[d * c.plane[0].sc[3]]);
      }
      dot = warp_sum(dot) * *kv8_scale(c.plane[0], page, kvh, row / c.group);
    }
    const float sc = kv8_score2(dot, p.scale, p.softcap);
    const float mn = fmaxf(m, sc);
    const float mu = mn == -INFINITY ? 0.f : mn;
    l = l * exp2f(m - mu) + exp2f(sc - mu);
    m = mn;
    if (vs == 0.f) continue;  // zero rows add to l only
    int ve;
    const float vm = frexpf(vs, &ve);
    if (!(fabsf(vs) < INFINITY)) ve = 0;
    if (rs == -INFINITY || (sc - rs) + (ve - re) > 0.f) {
      const float a = rs == -INFINITY ? 0.f : exp2f((rs - sc) + (re - ve));
      rs = sc;
      re = ve;
#pragma unroll
      for (int e = 0; e < kKv8MaxPerLane; ++e) acc[e] *= a;
    }
    const float e2 = (rs == -INFINITY ? 0.f : exp2f((sc - rs) + (ve - re))) * vm;
#pragma unroll
    for (int e = 0; e < kKv8MaxPerLane; ++e) {
      const int d = lane + 32 * e;
      if (d < c.D) acc[e] += e2 * Kv8<CODE>::dec(vr[d * c.plane[1].sc[3]]);
    }
  }
  __shared__ float sm_m[4], sm_l[4], sm_rs[4];
  __shared__ int sm_re[4];
  __shared__ float sm_o[4][32 * kKv8MaxPerLane];
  if (lane == 0) {
    sm_m[warp] = m;
    sm_l[warp] = l;
    sm_rs[warp] = rs;
    sm_re[warp] = re;
  }
#pragma unroll
  for (int e = 0; e < kKv8MaxPerLane; ++e) sm_o[warp][lane + 32 * e] = acc[e];
  __syncthreads();
  const float M = fmaxf(fmaxf(sm_m[0], sm_m[1]), fmaxf(sm_m[2], sm_m[3]));
  const float Mu = (M == -INFINITY) ? 0.f : M;
  float L = 0.f, f[4], RS = -INFINITY;
  int RE = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    L += sm_l[w] * exp2f(sm_m[w] - Mu);
    if (sm_rs[w] == -INFINITY) continue;
    if (RS == -INFINITY || (sm_rs[w] - RS) + (sm_re[w] - RE) > 0.f) {
      RS = sm_rs[w];
      RE = sm_re[w];
    }
  }
#pragma unroll
  for (int w = 0; w < 4; ++w) f[w] = sm_rs[w] == -INFINITY ? 0.f : exp2f((sm_rs[w] - RS) + (sm_re[w] - RE));
  // 2^(RS - M + RE), its whole part as an exponent
  const float diff = RS == -INFINITY ? 0.f : RS - Mu, whole = rintf(fmaxf(diff, -400.f));
  const float part = exp2f(fmaxf(diff, -400.f) - whole);
  T* out = static_cast<T*>(p.out) + s * p.so[0] + i * p.so[1] + h * p.so[2];
  for (int d = threadIdx.x; d < c.D; d += 128) {
    float o = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) o += sm_o[w][d] * f[w];
    // NaN scores give NaN, no key gives 0
    out[d * p.so[3]] = Elem<T>::from_f(L != 0.f ? ldexpf(o * part / L, static_cast<int>(whole) + RE) : 0.f);
  }
  if (threadIdx.x == 0) {
    const float lse2 = L != 0.f ? M + log2f(L) : -INFINITY;
    const int64_t at = (static_cast<int64_t>(s) * p.Lq + i) * p.H + h;
    if (p.lse) p.lse[at] = lse2 * kLn2;
    if (p.lse2) p.lse2[at] = lse2;
  }
}

template <typename T, int CODE>
__global__ void __launch_bounds__(128) kv8_weights_generic_kernel(const Kv8GenericParams p) {
  const Kv8View& c = p.c;
  const int kvh = blockIdx.y, s = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t ctx = min(static_cast<int64_t>(p.context_lens[s]), min(c.max_rows, p.width));
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * 4 + warp; r < ctx; r += 4 * static_cast<int64_t>(gridDim.x)) {
    const int64_t page = kv8_page(c, s, r);
    const int row = static_cast<int>(r % c.P);
    float kr[kKv8MaxPerLane];
#pragma unroll
    for (int e = 0; e < kKv8MaxPerLane; ++e) {
      const int d = lane + 32 * e;
      kr[e] = d < c.D && page >= 0 ? Kv8<CODE>::dec(kv8_row(c.plane[0], page, kvh, row)[d * c.plane[0].sc[3]]) : 0.f;
    }
    const float ks = page >= 0 ? *kv8_scale(c.plane[0], page, kvh, row / c.group) : 0.f;
    const int64_t full = min(static_cast<int64_t>(p.context_lens[s]), c.max_rows);
    float sum = 0.f;
    for (int i = 0; i < p.Lq; ++i) {
      if (r >= full - p.Lq + i + 1) continue;
      for (int g = 0; g < p.G; ++g) {
        const int h = kvh * p.G + g;
        const T* q = static_cast<const T*>(p.q) + s * p.sq[0] + i * p.sq[1] + h * p.sq[2];
        float dot = 0.f;
#pragma unroll
        for (int e = 0; e < kKv8MaxPerLane; ++e) {
          const int d = lane + 32 * e;
          if (d < c.D) dot += kr[e] * Elem<T>::to_f(q[d * p.sq[3]]);
        }
        dot = warp_sum(dot) * ks;
        sum += exp2f(kv8_score2(dot, p.scale, p.softcap) -
                     p.lse2[(static_cast<int64_t>(s) * p.Lq + i) * p.H + h]);
      }
    }
    if (lane == 0) p.weights[s * p.sw[0] + kvh * p.sw[1] + r * p.sw[2]] += sum;
  }
}

int kv8_attention_generic_launch(const Kv8View& c, const Kv8AttnArgs& a, cudaStream_t st) {
  Kv8GenericParams p{};
  p.c = c;
  p.q = a.q;
  p.out = a.out;
  for (int i = 0; i < 4; ++i) { p.sq[i] = a.sq[i]; p.so[i] = a.so[i]; }
  p.context_lens = a.context_lens;
  p.lse = a.lse;
  p.lse2 = a.weights ? static_cast<float*>(a.workspace) : nullptr;
  p.weights = a.weights;
  for (int i = 0; i < 3; ++i) p.sw[i] = a.sw[i];
  p.width = a.weights_width;
  p.H = a.H; p.Lq = a.Lq; p.G = a.H / c.Hkv;
  p.scale = a.scale;
  p.softcap = a.softcap;
  note_kernel("kv8_attention_generic");
  TAK_BY_DTYPE(a.dtype, TAK_BY_CODE(a.code_type, {
    kv8_attention_generic_kernel<T, CODE><<<dim3(a.H, a.Lq, c.num_seqs), 128, 0, st>>>(p);
    if (a.weights && a.weights_width > 0) {
      const int64_t keys = a.weights_width < c.max_rows ? a.weights_width : c.max_rows;
      const unsigned gx = static_cast<unsigned>(keys < 4 * 1024 ? (keys + 3) / 4 : 1024);
      if (gx) kv8_weights_generic_kernel<T, CODE><<<dim3(gx, c.Hkv, c.num_seqs), 128, 0, st>>>(p);
    }
  }));
  return 0;
}

}  // namespace tak
