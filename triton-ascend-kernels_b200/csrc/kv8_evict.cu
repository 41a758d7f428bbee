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
#include <cooperative_groups.h>

#include <cstdio>

#include "kv8.cuh"

namespace tak {

namespace cg = cooperative_groups;

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

// Selection with the weights in registers: a cluster of CTAs holds one (sequence,
// head), KPT weights a thread.  The threshold key is found two bits at a time: the
// three candidates for the next two bits are counted in one pass over the
// registers (three ten-bit counts in one warp reduction), summed over the cluster
// through distributed shared memory.  A histogram instead would serialise on
// shared-memory atomics: weights of one sequence share few exponents.
template <int KPT>
__global__ void __launch_bounds__(kSelThreads) kv8_evict_select_reg_kernel(const Kv8EvictParams p) {
  cg::cluster_group cluster = cg::this_cluster();
  const int cs = cluster.num_blocks(), rank = cluster.block_rank();
  const int h = blockIdx.x / cs, s = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = kv8_evict_rows(p, s), m = min(n, p.budget);
  int32_t* kept = p.kept + (static_cast<int64_t>(s) * p.c.Hkv + h) * p.budget;
  const int all = cs * kSelThreads, at = rank * kSelThreads + tid;
  if (h == 0 && at == 0) p.new_lens[s] = m;
  for (int j = m + at; j < p.budget; j += all) kept[j] = -1;
  if (n <= p.budget) {
    for (int j = at; j < n; j += all) kept[j] = j;
    return;
  }
  float* w = p.weights + s * p.sw[0] + h * p.sw[1];
  const int64_t ws = p.sw[2];
  const int cand = n - p.recent, take = p.budget - p.recent;
  const int base = rank * KPT * kSelThreads;  // the CTA's first position

  __shared__ uint32_t warp_part[2][32];       // [parity] packed counts of the warps
  __shared__ uint32_t cta_part[2][3];         // [parity] the CTA's counts, read by the cluster
  __shared__ uint32_t cnt[KPT * 32];          // kept (low half) and tied (high half) keys of each warp's 32
  __shared__ uint32_t scan_part[32];
  __shared__ uint2 cta_total;                 // kept, tied keys of the CTA

  // keys of positions past the candidates are 0 and are told apart by position
  float val[KPT];
  uint32_t key[KPT];
#pragma unroll
  for (int k = 0; k < KPT; ++k) {
    const int i = base + k * kSelThreads + tid;
    val[k] = i < n ? w[i * ws] : 0.f;
  }
#pragma unroll
  for (int k = 0; k < KPT; ++k) key[k] = base + k * kSelThreads + tid < cand ? weight_key(val[k]) : 0u;

  // largest T with at least `take` candidate keys >= T; key 0 (only a negative
  // NaN's, which weight_key does not give) stands for no candidate
  uint32_t T = 0;
  if (take > 0) {
    for (int shift = 30, it = 0; shift >= 0; shift -= 2, ++it) {
      const uint32_t t1 = T | (1u << shift), t2 = T | (2u << shift), t3 = T | (3u << shift);
      uint32_t c = 0;
#pragma unroll
      for (int k = 0; k < KPT; ++k)
        c += (key[k] >= t1 ? 1u : 0u) + (key[k] >= t2 ? 1u << 10 : 0u) + (key[k] >= t3 ? 1u << 20 : 0u);
      c = __reduce_add_sync(0xffffffffu, c);
      if (lane == 0) warp_part[it & 1][warp] = c;
      __syncthreads();
      uint32_t total[3] = {0, 0, 0};
      const uint32_t q = warp_part[it & 1][lane];
#pragma unroll
      for (int x = 0; x < 3; ++x) total[x] = __reduce_add_sync(0xffffffffu, (q >> (10 * x)) & 1023u);
      if (cs > 1) {
        if (tid < 3) cta_part[it & 1][tid] = tid == 0 ? total[0] : tid == 1 ? total[1] : total[2];
        cluster.sync();
#pragma unroll
        for (int x = 0; x < 3; ++x) {
          const uint32_t v = lane < cs ? *cluster.map_shared_rank(&cta_part[it & 1][x], lane) : 0u;
          total[x] = __reduce_add_sync(0xffffffffu, v);
        }
      }
      const uint32_t need = static_cast<uint32_t>(take);
      T = total[2] >= need ? t3 : total[1] >= need ? t2 : total[0] >= need ? t1 : T;
    }
  } else {
    T = 0xffffffffu;
  }

  // kept: the recent rows and keys above T; tied: keys equal to T, of which the
  // first (take - keys above) stay
  uint32_t gt[KPT], eq[KPT];
#pragma unroll
  for (int k = 0; k < KPT; ++k) {
    const int i = base + k * kSelThreads + tid;
    const bool is_gt = (i >= cand && i < n) || (take > 0 && i < cand && key[k] > T);
    const bool is_eq = take > 0 && i < cand && key[k] == T;
    gt[k] = __ballot_sync(0xffffffffu, is_gt);
    eq[k] = __ballot_sync(0xffffffffu, is_eq);
    if (lane == 0) cnt[k * 32 + warp] = __popc(gt[k]) | (__popc(eq[k]) << 16);
  }
  __syncthreads();
  // exclusive scan of cnt (KPT * 32 <= 512 entries; sums stay below 2^16)
  {
    uint32_t v = tid < KPT * 32 ? cnt[tid] : 0u, x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += u;
    }
    if (lane == 31) scan_part[warp] = x;
    __syncthreads();
    uint32_t y = scan_part[lane], z = y;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, z, o);
      if (lane >= o) z += u;
    }
    const uint32_t before = __shfl_sync(0xffffffffu, z - y, warp);
    if (tid < KPT * 32) cnt[tid] = before + x - v;
    if (tid == kSelThreads - 1) cta_total = make_uint2((before + x) & 0xffffu, (before + x) >> 16);
  }
  __syncthreads();
  cluster.sync();  // totals are there; and every weight of the cluster is in registers
  uint32_t gt0 = 0, eq0 = 0, gt_all = 0;
  for (int r = 0; r < cs; ++r) {
    const uint2 t = *cluster.map_shared_rank(&cta_total, r);
    if (r < rank) { gt0 += t.x; eq0 += t.y; }
    gt_all += t.x;
  }
  const uint32_t ties = static_cast<uint32_t>(p.budget) - gt_all;  // how many tied keys stay
  const uint32_t below = (1u << lane) - 1;
#pragma unroll
  for (int k = 0; k < KPT; ++k) {
    const uint32_t c = cnt[k * 32 + warp];
    const uint32_t g_before = gt0 + (c & 0xffffu) + __popc(gt[k] & below);
    const uint32_t e_before = eq0 + (c >> 16) + __popc(eq[k] & below);
    const bool is_gt = (gt[k] >> lane) & 1, is_eq = (eq[k] >> lane) & 1;
    if (is_gt || (is_eq && e_before < ties)) {
      const uint32_t j = g_before + min(e_before, ties);
      kept[j] = base + k * kSelThreads + tid;
      w[j * ws] = val[k];
    }
  }
  for (int i = m + at; i < n; i += all) w[i * ws] = 0.f;
  cluster.sync();  // no CTA leaves while another reads its totals
}

// Moves the kept rows of one (sequence, head, K or V).  A cluster moves `cs`
// windows of rows at a step: sources of a step lie at or after it, so the next
// step's rows are fetched (cp.async) while this one's are written, and one cluster
// barrier a step keeps every read before the writes that reach it.
template <int CODE, int VEC>
__global__ void __launch_bounds__(256) kv8_evict_move_kernel(const Kv8EvictParams p) {
  extern __shared__ __align__(16) uint8_t stage[];  // [2][window][D] codes, then the scales
  cg::cluster_group cluster = cg::this_cluster();
  const Kv8View& c = p.c;
  const int cs = cluster.num_blocks(), rank = cluster.block_rank();
  const int h = blockIdx.x / cs, s = blockIdx.y, tid = threadIdx.x, D = c.D, pieces = D / VEC;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the selection
  const Kv8Plane& pl = c.plane[blockIdx.z];
  const int n = kv8_evict_rows(p, s);
  if (n <= p.budget) return;
  const int m = p.budget, win = p.window;
  const int32_t* kept = p.kept + (static_cast<int64_t>(s) * c.Hkv + h) * p.budget;
  float* was = reinterpret_cast<float*>(stage + 2 * static_cast<size_t>(win) * D);  // [2][win] scales of the rows
  float* now = was + 2 * win;                                                       // [win] of the groups, then
  const uint8_t** src = reinterpret_cast<const uint8_t**>(now + win);               // [win] row addresses
  uint8_t** dst = const_cast<uint8_t**>(src + win);                                 // [win]

  auto fetch = [&](int j0, int buf) {  // a window's rows and scales; a row outside the cache is zeros
    const int rows = min(win, m - j0);
    for (int r = tid; r < rows; r += 256) {
      const int i = kept[j0 + r];
      const int64_t page = kv8_page(c, s, i);
      const int row = i % c.P;
      src[r] = page >= 0 ? kv8_row(pl, page, h, row) : nullptr;
      was[buf * win + r] = page >= 0 ? *kv8_scale(pl, page, h, row / c.group) : 0.f;
    }
    __syncthreads();
    uint8_t* to = stage + static_cast<size_t>(buf) * win * D;
    for (int e = tid; e < rows * pieces; e += 256) {
      const int r = e / pieces, d = (e - r * pieces) * VEC;
      if (VEC == 16) {
        cp_async_16(to + r * D + d, src[r] ? src[r] + d : pl.code, src[r] != nullptr);
      } else {
        to[r * D + d] = src[r] ? src[r][d * pl.sc[3]] : 0;
      }
    }
  };
  const int step = cs * win;
  fetch(min(rank * win, m), 0);
  cp_async_wait_all();
  cluster.sync();
  for (int j0 = rank * win, buf = 0; j0 - rank * win < m; j0 += step, buf ^= 1) {
    const int rows = max(0, min(win, m - j0));
    __syncthreads();  // the row addresses of the last fetch have been used
    if (j0 + step < m) fetch(j0 + step, buf ^ 1);
    const float* ws = was + buf * win;
    for (int r = tid; r < rows; r += 256) {
      const int64_t page = kv8_page(c, s, j0 + r);
      const int row = (j0 + r) % c.P;
      dst[r] = page >= 0 ? kv8_row(pl, page, h, row) : nullptr;
      if (r % c.group == 0) {
        float big = 0.f;
        for (int x = r; x < min(rows, r + c.group); ++x) big = kv8_scale_max(big, ws[x]);
        now[r / c.group] = big;
        if (page >= 0) *kv8_scale(pl, page, h, row / c.group) = big;
      }
    }
    __syncthreads();
    const uint8_t* from = stage + static_cast<size_t>(buf) * win * D;
    for (int e = tid; e < rows * pieces; e += 256) {
      const int r = e / pieces, d = (e - r * pieces) * VEC;
      if (dst[r] == nullptr) continue;
      const float a = ws[r], b = now[r / c.group];
      if (VEC == 16) {
        uint4 q = *reinterpret_cast<const uint4*>(from + r * D + d);
        if (a < b) {
          const float ratio = a / b;
          q.x = kv8_rescale4<CODE>(q.x, ratio);
          q.y = kv8_rescale4<CODE>(q.y, ratio);
          q.z = kv8_rescale4<CODE>(q.z, ratio);
          q.w = kv8_rescale4<CODE>(q.w, ratio);
        }
        *reinterpret_cast<uint4*>(dst[r] + d) = q;
      } else {
        uint8_t q = from[r * D + d];
        if (a < b) q = Kv8<CODE>::enc(Kv8<CODE>::dec(q) * (a / b));
        dst[r][d * pl.sc[3]] = q;
      }
    }
    cp_async_wait_all();
    cluster.sync();
  }
}

// launch with a cluster, optionally as a programmatic dependent of the last grid
template <typename K, typename... A>
static int launch_cluster(K kern, dim3 grid, int threads, size_t smem, int cs, bool dependent, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cs;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  if (e == cudaSuccess) return 0;
  char buf[160];
  std::snprintf(buf, sizeof(buf), "kv8 evict: launch failed: %s", cudaGetErrorString(e));
  return set_error(3, buf);
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
  // ---- selection: in registers up to 8 CTAs x 1024 threads x 16 weights ----
  const int64_t rows = width < c.max_rows ? width : c.max_rows;
  const int64_t sel = kSelThreads;
  note_kernel("kv8_evict");
  if (rows <= 16 * 8 * sel) {
    int cs = 1;
    while (rows > 16 * sel * cs) cs *= 2;
    const dim3 grid(c.Hkv * cs, c.num_seqs);
    int r;
    if (rows <= 4 * sel) r = launch_cluster(kv8_evict_select_reg_kernel<4>, grid, kSelThreads, 0, cs, false, st, p);
    else if (rows <= 8 * sel) r = launch_cluster(kv8_evict_select_reg_kernel<8>, grid, kSelThreads, 0, cs, false, st, p);
    else r = launch_cluster(kv8_evict_select_reg_kernel<16>, grid, kSelThreads, 0, cs, false, st, p);
    if (r) return r;
  } else {
    kv8_evict_select_kernel<<<dim3(c.Hkv, c.num_seqs), kSelThreads, 0, st>>>(p);
  }
  // ---- move: windows of about 32 KB of rows, a multiple of the group ----
  int64_t win = 32768 / c.D / c.group * c.group;
  if (win < c.group) win = c.group;
  if (win > 256) win = 256 / c.group * c.group;
  p.window = static_cast<int>(win);
  const int64_t smem = 2 * win * c.D + 3 * win * 4 + 2 * win * 8 + 16;
  if (smem > 200 * 1024) return set_error(2, "kv8 evict: group * head_dim is too large");
  // a cluster per (sequence, head, K or V) where there are fewer of them than SMs
  const int64_t units = 2 * static_cast<int64_t>(c.Hkv) * c.num_seqs;
  int cs = 1;
  while (cs < 8 && units * cs < 2 * num_sms() && cs * win < budget) cs *= 2;
  bool vec = c.D % 16 == 0;
  for (const Kv8Plane& pl : c.plane)
    vec = vec && pl.sc[3] == 1 && (reinterpret_cast<uintptr_t>(pl.code) & 15) == 0 && ((pl.sc[0] | pl.sc[1] | pl.sc[2]) & 15) == 0;
  TAK_BY_CODE(code_type, {
    auto kern = vec ? kv8_evict_move_kernel<CODE, 16> : kv8_evict_move_kernel<CODE, 1>;
    if (const int r = ensure_smem_attr(reinterpret_cast<const void*>(kern), static_cast<int>(smem))) return r;
    return launch_cluster(kern, dim3(c.Hkv * cs, c.num_seqs, 2), 256, static_cast<size_t>(smem), cs, true, st, p);
  });
  return 0;
}

}  // namespace tak
