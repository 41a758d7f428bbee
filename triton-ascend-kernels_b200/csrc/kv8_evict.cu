// Eviction from the 8-bit KV cache by accumulated attention weight.
//
// For each (sequence, KV head) with n > budget rows: the last `recent` rows
// stay, and of the others the budget - recent with the largest accumulated
// weight (ties to the lowest position, NaN above every number).  Kept rows
// move to the front of the sequence in ascending order, in place.  A group of
// the compacted rows takes the largest scale of the rows that it receives;
// a row that came under a smaller one is requantised,
//   code' = round(code * (its scale / the group's scale)),
// and a row whose scale is the group's keeps its codes.
#include "kv8.cuh"

namespace tak {

struct Kv8EvictParams {
  Kv8View c;
  const int32_t* context_lens;
  float* weights; int64_t sw[3];
  int64_t width;
  int budget, recent;
  int32_t* kept;      // [B, Hkv, budget]
  int32_t* new_lens;  // [B]
  int window;         // rows moved at a time, a multiple of group
};

__device__ __forceinline__ int kv8_evict_rows(const Kv8EvictParams& p, int s) {
  const int64_t n = min(static_cast<int64_t>(p.context_lens[s]), min(p.width, p.c.max_rows));
  return n > 0 ? static_cast<int>(n) : 0;
}

// unsigned key ordered as the floats are: -0 equals +0, NaN on top
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t b = __float_as_uint(w + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

constexpr int kSelThreads = 1024;

// inclusive scan of (a, b) over the block; returns the exclusive parts and
// leaves the block totals in tot
__device__ __forceinline__ uint2 block_scan2(uint32_t a, uint32_t b, uint2* part, uint2& tot) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t x = a, y = b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t u = __shfl_up_sync(0xffffffffu, x, o), v = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o) { x += u; y += v; }
  }
  if (lane == 31) part[warp] = make_uint2(x, y);
  __syncthreads();
  if (warp == 0) {
    uint2 w = part[lane];
    uint32_t u = w.x, v = w.y;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t uu = __shfl_up_sync(0xffffffffu, u, o), vv = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) { u += uu; v += vv; }
    }
    part[lane] = make_uint2(u, v);
  }
  __syncthreads();
  const uint2 before = warp ? part[warp - 1] : make_uint2(0, 0);
  tot = part[31];
  __syncthreads();
  return make_uint2(before.x + x - a, before.y + y - b);
}

__global__ void __launch_bounds__(kSelThreads) kv8_evict_select_kernel(const Kv8EvictParams p) {
  const int h = blockIdx.x, s = blockIdx.y, tid = threadIdx.x;
  const int n = kv8_evict_rows(p, s), m = min(n, p.budget);
  int32_t* kept = p.kept + (static_cast<int64_t>(s) * p.c.Hkv + h) * p.budget;
  if (h == 0 && tid == 0) p.new_lens[s] = m;
  for (int j = m + tid; j < p.budget; j += kSelThreads) kept[j] = -1;
  if (n <= p.budget) {
    for (int j = tid; j < n; j += kSelThreads) kept[j] = j;
    return;
  }
  float* w = p.weights + s * p.sw[0] + h * p.sw[1];
  const int64_t ws = p.sw[2];
  const int cand = n - p.recent, take = p.budget - p.recent;

  // threshold: the take-th largest key of the candidates, digit by digit
  __shared__ uint32_t hist[256];
  __shared__ uint32_t sh_prefix, sh_left;
  __shared__ uint2 part[32];
  uint32_t prefix = 0, left = take;  // keys above the threshold's digits so far are already counted out of `left`
  for (int shift = 24; take > 0 && shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int i = tid; i < cand; i += kSelThreads) {
      const uint32_t key = weight_key(w[i * ws]);
      if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(key >> shift) & 255], 1u);
    }
    __syncthreads();
    if (tid == 0) {
      uint32_t l = left;
      int d = 255;
      while (d > 0 && hist[d] < l) l -= hist[d--];
      sh_prefix = prefix | (static_cast<uint32_t>(d) << shift);
      sh_left = l;
    }
    __syncthreads();
    prefix = sh_prefix;
    left = sh_left;
  }
  const uint32_t cut = take > 0 ? prefix : 0xffffffffu;  // keys above it stay, and the first `ties` equal to it
  const uint32_t ties = take > 0 ? left : 0;

  // stable compaction of indices and weights (in place: a row's new place is
  // never after its old one, and a tile is read before it is written)
  uint32_t base_gt = 0, base_eq = 0;
  for (int t0 = 0; t0 < n; t0 += kSelThreads) {
    const int i = t0 + tid;
    float v = 0.f;
    uint32_t gt = 0, eq = 0;
    if (i < n) {
      v = w[i * ws];
      if (i >= cand) {
        gt = 1;
      } else {
        const uint32_t key = weight_key(v);
        gt = key > cut;
        eq = key == cut && ties > 0;
      }
    }
    uint2 tot;
    const uint2 ex = block_scan2(gt, eq, part, tot);
    const uint32_t eq_before = base_eq + ex.y;
    if (gt || (eq && eq_before < ties)) {
      const uint32_t j = base_gt + ex.x + min(eq_before, ties);
      kept[j] = i;
      w[j * ws] = v;
    }
    base_gt += tot.x;
    base_eq += tot.y;
  }
  __syncthreads();
  for (int i = m + tid; i < n; i += kSelThreads) w[i * ws] = 0.f;
}

// Moves the kept rows of one (sequence, head, K or V), a window of rows at a
// time: sources of a window lie at or after it, so once a window has been read
// it may be written.
template <int CODE>
__global__ void __launch_bounds__(256) kv8_evict_move_kernel(const Kv8EvictParams p) {
  extern __shared__ __align__(16) uint8_t stage[];  // [window][D] codes
  const Kv8View& c = p.c;
  const int h = blockIdx.x, s = blockIdx.y, tid = threadIdx.x, D = c.D;
  const Kv8Plane& pl = c.plane[blockIdx.z];
  const int n = kv8_evict_rows(p, s);
  if (n <= p.budget) return;
  const int m = p.budget;
  const int32_t* kept = p.kept + (static_cast<int64_t>(s) * c.Hkv + h) * p.budget;
  float* was = reinterpret_cast<float*>(stage + static_cast<size_t>(p.window) * D);  // [window]
  float* now = was + p.window;                                                       // [window / group]
  for (int j0 = 0; j0 < m; j0 += p.window) {
    const int rows = min(p.window, m - j0);
    for (int r = tid; r < rows; r += 256) {
      const int src = kept[j0 + r];
      const int64_t page = kv8_page(c, s, src);
      was[r] = page >= 0 ? *kv8_scale(pl, page, h, src % c.P / c.group) : 0.f;
    }
    for (int e = tid; e < rows * D; e += 256) {
      const int src = kept[j0 + e / D];
      const int64_t page = kv8_page(c, s, src);
      stage[e] = page >= 0 ? kv8_row(pl, page, h, src % c.P)[(e % D) * pl.sc[3]] : 0;
    }
    __syncthreads();
    for (int g = tid; g * c.group < rows; g += 256) {
      float big = 0.f;
      for (int r = g * c.group; r < min(rows, (g + 1) * c.group); ++r) big = kv8_scale_max(big, was[r]);
      now[g] = big;
      const int64_t page = kv8_page(c, s, j0 + g * c.group);
      if (page >= 0) *kv8_scale(pl, page, h, (j0 + g * c.group) % c.P / c.group) = big;
    }
    __syncthreads();
    for (int e = tid; e < rows * D; e += 256) {
      const int r = e / D;
      const int64_t page = kv8_page(c, s, j0 + r);
      if (page < 0) continue;
      const float a = was[r], b = now[r / c.group];
      uint8_t q = stage[e];
      if (a < b) q = Kv8<CODE>::enc(Kv8<CODE>::dec(q) * (a / b));
      kv8_row(pl, page, h, (j0 + r) % c.P)[(e % D) * pl.sc[3]] = q;
    }
    __syncthreads();
  }
}

int kv8_evict_launch(const Kv8View& c, int code_type, const int32_t* context_lens, float* weights,
                     const int64_t* sw, int64_t width, int64_t budget, int64_t recent, int32_t* kept,
                     int32_t* new_lens, cudaStream_t st) {
  Kv8EvictParams p{};
  p.c = c;
  p.context_lens = context_lens;
  p.weights = weights;
  for (int i = 0; i < 3; ++i) p.sw[i] = sw[i];
  p.width = width;
  p.budget = static_cast<int>(budget);
  p.recent = static_cast<int>(recent);
  p.kept = kept;
  p.new_lens = new_lens;
  p.window = c.group * (c.group < 64 ? 64 / c.group : 1);
  const int64_t smem = static_cast<int64_t>(p.window) * (c.D + 4) + (p.window / c.group + 4) * 4;
  if (smem > 200 * 1024) return set_error(2, "kv8 evict: group * head_dim is too large");
  note_kernel("kv8_evict");
  kv8_evict_select_kernel<<<dim3(c.Hkv, c.num_seqs), kSelThreads, 0, st>>>(p);
  TAK_BY_CODE(code_type, {
    auto kern = kv8_evict_move_kernel<CODE>;
    if (const int r = ensure_smem_attr(reinterpret_cast<const void*>(kern), static_cast<int>(smem))) return r;
    kern<<<dim3(c.Hkv, c.num_seqs, 2), 256, smem, st>>>(p);
  });
  return 0;
}

}  // namespace tak
