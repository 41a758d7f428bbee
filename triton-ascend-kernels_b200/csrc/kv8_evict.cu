// Eviction from the 8-bit KV cache by accumulated attention weight.
//
// For each (sequence, KV head) with n > budget rows: the last `recent` rows
// stay, and of the others the budget - recent with the largest accumulated
// weight (ties to the lowest position, NaN above every number; rows past the end of
// `weights` have accumulated none and weigh 0).  Kept rows
// move to the front of the sequence in ascending order, in place.  A group of
// the compacted rows takes the largest scale of the rows that it receives;
// a row that came under a smaller one is requantised,
//   code' = round(code * (its scale / the group's scale)),
// and a row whose scale is the group's keeps its codes.
#include <cooperative_groups.h>

#include <cstdio>
#include <map>
#include <mutex>
#include <tuple>

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
  int stages;         // windows in shared memory: 2, or 1 where two do not fit
};

__device__ __forceinline__ int kv8_evict_rows(const Kv8EvictParams& p, int s) {
  const int64_t n = min(static_cast<int64_t>(p.context_lens[s]), p.c.max_rows);
  return n > 0 ? static_cast<int>(n) : 0;
}
constexpr uint32_t kZeroKey = 0x80000000u;  // weight_key(0)

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

// Selection for sequences too long for the registers of a cluster (where table and
// weights both pass 131072 rows): one CTA per (sequence, head) that reads its weights
// once for each of four eight-bit digits and once more to compact them.  Bound by that
// CTA's latency: 8 heads of 131073 weights in 314 us, of 262144 in 608, of 4096 in such
// a table in 29.
__global__ void __launch_bounds__(kSelThreads) kv8_evict_select_kernel(const Kv8EvictParams p) {
  const int h = blockIdx.x, s = blockIdx.y, tid = threadIdx.x;
  const int n = kv8_evict_rows(p, s), m = min(n, p.budget);
  int32_t* kept = p.kept + (static_cast<int64_t>(s) * p.c.Hkv + h) * p.budget;
  if (h == 0 && tid == 0) p.new_lens[s] = m;
  // (unsigned: with a budget near 2^31 the last step passes it)
  for (uint32_t j = m + tid; j < static_cast<uint32_t>(p.budget); j += kSelThreads) kept[j] = -1;
  if (n <= p.budget) {
    for (int j = tid; j < n; j += kSelThreads) kept[j] = j;
    return;
  }
  float* w = p.weights + s * p.sw[0] + h * p.sw[1];
  const int64_t ws = p.sw[2];
  const int cand = n - p.recent, take = p.budget - p.recent;
  const int nw = static_cast<int>(min(static_cast<int64_t>(n), p.width));  // rows that have a weight

  // threshold: the take-th largest key of the candidates, digit by digit
  __shared__ uint32_t hist[256];
  __shared__ uint32_t sh_prefix, sh_left;
  __shared__ uint2 part[32];
  uint32_t prefix = 0, left = take;  // keys above the threshold's digits so far are already counted out of `left`
  for (int shift = 24; take > 0 && shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int i = tid; i < cand; i += kSelThreads) {
      const uint32_t key = i < nw ? weight_key(w[i * ws]) : kZeroKey;
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
      if (i < nw) v = w[i * ws];
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
      if (j < nw) w[j * ws] = v;
    }
    base_gt += tot.x;
    base_eq += tot.y;
  }
  __syncthreads();
  for (int i = m + tid; i < nw; i += kSelThreads) w[i * ws] = 0.f;
}

// Selection with the weights in registers: a cluster of CTAs holds one (sequence,
// head), KPT weights a thread.  The threshold key is found digit by digit (11, 11
// and 10 bits): each CTA counts its keys in shared memory, the cluster's counts are
// added through distributed shared memory, and every CTA finds the digit in which
// the take-th largest key lies.  Bound by latency, the cluster barriers and the rounds
// through distributed shared memory: 8 heads of 100000 weights in 28 us, 48 x 8 heads
// of up to 8192 in 22.  (Counting two bits at a time in registers, 16 cluster barriers
// instead of three, took 75 us for 8 heads of 100000 weights; eight weights a thread in
// clusters of 16, 56.)
//
// Rows past the end of `weights` are not held: they are one run of keys of weight 0
// after all others, so their number goes into the counts, and the kept ones among them
// follow the held rows in order.
constexpr int kBins = 2048;

template <int KPT>
__global__ void __launch_bounds__(kSelThreads, KPT <= 8 ? 2 : 1) kv8_evict_select_reg_kernel(const Kv8EvictParams p) {
  cg::cluster_group cluster = cg::this_cluster();
  const int cs = cluster.num_blocks(), rank = cluster.block_rank();
  const int h = blockIdx.x / cs, s = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int n = kv8_evict_rows(p, s), m = min(n, p.budget);
  int32_t* kept = p.kept + (static_cast<int64_t>(s) * p.c.Hkv + h) * p.budget;
  const int all = cs * kSelThreads, at = rank * kSelThreads + tid;
  if (h == 0 && at == 0) p.new_lens[s] = m;
  // (unsigned: with a budget near 2^31 the last step passes it)
  for (uint32_t j = m + at; j < static_cast<uint32_t>(p.budget); j += all) kept[j] = -1;
  if (n <= p.budget) {
    for (int j = at; j < n; j += all) kept[j] = j;
    return;
  }
  float* w = p.weights + s * p.sw[0] + h * p.sw[1];
  const int64_t ws = p.sw[2];
  const int cand = n - p.recent, take = p.budget - p.recent;
  const int nw = static_cast<int>(min(static_cast<int64_t>(n), p.width));  // rows that have a weight
  const int held = min(cand, nw), bare = cand - held;                      // candidates that have one, and the others
  const int base = rank * KPT * kSelThreads;  // the CTA's first position

  __shared__ uint32_t hist[3][kBins];         // one per digit: no barrier to clear them between
  __shared__ uint32_t cnt[KPT * 32];          // kept (low half) and tied (high half) keys of each warp's 32
  __shared__ uint32_t scan_part[32];
  __shared__ uint32_t sh_digit, sh_left;
  __shared__ uint2 cta_total;                 // kept, tied keys of the CTA

  auto everyone = [&]() {
    if (cs > 1) cluster.sync(); else __syncthreads();
  };

  float val[KPT];
#pragma unroll
  for (int k = 0; k < KPT; ++k) {
    const int i = base + k * kSelThreads + tid;
    val[k] = i < nw ? w[i * ws] : 0.f;
  }
  for (int i = tid; i < 3 * kBins; i += kSelThreads) hist[0][i] = 0;
  __syncthreads();

  uint32_t T = 0, left = take;  // digits found so far; how many of the keys that have them stay
#pragma unroll
  for (int d = 0; d < 3; ++d) {
    if (take == 0) break;
    const int shift = d == 0 ? 21 : d == 1 ? 10 : 0;
    const uint32_t bins = d == 2 ? 1024 : 2048;
#pragma unroll
    for (int k = 0; k < KPT; ++k) {
      const int i = base + k * kSelThreads + tid;
      const uint32_t key = weight_key(val[k]);
      if (i < held && (d == 0 || (key >> (d == 1 ? 21 : 10)) == (T >> (d == 1 ? 21 : 10))))
        atomicAdd(&hist[d][(key >> shift) & (bins - 1)], 1u);
    }
    if (at == 0 && bare > 0 && (d == 0 || (kZeroKey >> (d == 1 ? 21 : 10)) == (T >> (d == 1 ? 21 : 10))))
      atomicAdd(&hist[d][(kZeroKey >> shift) & (bins - 1)], static_cast<uint32_t>(bare));
    everyone();
    // bins from the top: thread t has bins - 1 - 2 t and the one below
    uint32_t c0 = 0, c1 = 0;
    const int top = static_cast<int>(bins) - 1 - 2 * tid;
    if (top > 0) {
#pragma unroll
      for (int r = 0; r < 8; ++r) {  // at most 8 CTAs: all the reads in flight at once
        if (r >= cs) break;
        const uint2 v = *reinterpret_cast<const uint2*>(cluster.map_shared_rank(&hist[d][top - 1], r));
        c0 += v.y;
        c1 += v.x;
      }
    }
    uint32_t x = c0 + c1;
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
    const uint32_t before = __shfl_sync(0xffffffffu, z - y, warp) + x - c0 - c1;  // keys in higher bins
    if (before < left && left <= before + c0 + c1) {
      const bool second = left > before + c0;
      sh_digit = top - (second ? 1 : 0);
      sh_left = left - before - (second ? c0 : 0u);
    }
    __syncthreads();
    T |= sh_digit << shift;
    left = sh_left;
  }
  if (take == 0) T = 0xffffffffu;
  const uint32_t ties = take > 0 ? left : 0;  // how many of the keys equal to T stay

  // kept: the recent rows and keys above T; tied: keys equal to T
#pragma unroll
  for (int k = 0; k < KPT; ++k) {
    const int i = base + k * kSelThreads + tid;
    const uint32_t key = weight_key(val[k]);
    const unsigned gt = __ballot_sync(0xffffffffu, (i >= cand && i < nw) || (i < held && key > T));
    const unsigned eq = __ballot_sync(0xffffffffu, i < held && key == T && ties > 0);
    if (lane == 0) cnt[k * 32 + warp] = __popc(gt) | (__popc(eq) << 16);
  }
  __syncthreads();
  // exclusive scan of cnt (KPT * 32 <= 512 entries; sums stay below 2^16)
  {
    const uint32_t v = tid < KPT * 32 ? cnt[tid] : 0u;
    uint32_t x = v;
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
  everyone();  // totals are there; and every weight of the cluster is in registers
  uint32_t gt0 = 0, eq0 = 0;
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    if (r >= rank) break;
    const uint2 t = *cluster.map_shared_rank(&cta_total, r);
    gt0 += t.x;
    eq0 += t.y;
  }
  const uint32_t below = (1u << lane) - 1;
#pragma unroll
  for (int k = 0; k < KPT; ++k) {
    const int i = base + k * kSelThreads + tid;
    const uint32_t key = weight_key(val[k]), c = cnt[k * 32 + warp];
    const bool is_gt = (i >= cand && i < nw) || (i < held && key > T), is_eq = i < held && key == T && ties > 0;
    const uint32_t g_before = gt0 + (c & 0xffffu) + __popc(__ballot_sync(0xffffffffu, is_gt) & below);
    const uint32_t e_before = eq0 + (c >> 16) + __popc(__ballot_sync(0xffffffffu, is_eq) & below);
    if (is_gt || (is_eq && e_before < ties)) {
      const uint32_t j = g_before + min(e_before, ties);
      kept[j] = i;
      w[j * ws] = val[k];
    }
  }
  if (n > nw) {  // rows without a weight: the first `more` of the candidates, and the recent ones
    uint32_t gts = 0, eqs = 0;
    for (int r = 0; r < cs; ++r) {
      const uint2 t = *cluster.map_shared_rank(&cta_total, r);
      gts += t.x;
      eqs += t.y;
    }
    const int front = static_cast<int>(gts + min(eqs, ties));
    const int more = kZeroKey > T ? bare : kZeroKey == T ? static_cast<int>(ties - min(eqs, ties)) : 0;
    for (int j = front + at; j < m; j += all) {
      const int b = j - front;
      kept[j] = b < more ? held + b : max(cand, nw) + (b - more);
      if (j < nw) w[j * ws] = 0.f;
    }
  }
  for (int i = m + at; i < nw; i += all) w[i * ws] = 0.f;
  everyone();  // no CTA leaves while another reads its totals
}

// Moves the kept rows of one (sequence, head, K or V).  A cluster moves `cs`
// windows of rows at a step: sources of a step lie at or after it, so the next
// step's rows are fetched (cp.async) while this one's are written, and one cluster
// barrier a step keeps every read before the writes that reach it.  Thread r looks
// after row r of the windows: its position is read three steps ahead, its page two,
// its scale one, so that no step waits for a chain of loads.
//
// Bound by the issue slots of the requantisation and the row lookups (57 % issue),
// then by memory: 36 x 8 heads x 2048 rows of 128, K and V, in 75 us (302 MB moved,
// 4.0 TB/s, 61 % of the measured copy rate; 66 us over a cache that an eviction has
// compacted, where no row changes its scale); one sequence's 8 heads x 16384 rows, over
// clusters of 16, in 26.  Windows of 16 KB took 14 % longer.  Pieces held in registers
// so that four CTAs fit an SM: 10 % less where that saves a wave, 25 % more elsewhere.
template <int CODE, int VEC>
__global__ void __launch_bounds__(256) kv8_evict_move_kernel(const __grid_constant__ Kv8EvictParams p) {
  extern __shared__ __align__(16) uint8_t stage[];  // [stages][window][D] codes, then per row:
  cg::cluster_group cluster = cg::this_cluster();
  const Kv8View& c = p.c;
  const int cs = cluster.num_blocks(), rank = cluster.block_rank();
  const int h = blockIdx.x / cs, s = blockIdx.y, tid = threadIdx.x, D = c.D, pieces = D / VEC;
  const Kv8Plane pl = blockIdx.z ? c.plane[1] : c.plane[0];
  const int win = p.window;
  const int flip = p.stages - 1;  // step w uses stage w & flip
  const uint8_t** src = reinterpret_cast<const uint8_t**>(stage + (p.stages * static_cast<size_t>(win) * D + 15) / 16 * 16);  // [2][win]
  struct alignas(16) Dst { uint8_t* row; float ratio; };
  Dst* dst = reinterpret_cast<Dst*>(const_cast<uint8_t**>(src + 2 * win));                           // [win]
  float* was = reinterpret_cast<float*>(dst + win);                                                  // [win] scales
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the selection
  const int n = kv8_evict_rows(p, s);
  if (n <= p.budget) return;
  const int m = p.budget, step = cs * win, first = rank * win;
  const int32_t* kept = p.kept + (static_cast<int64_t>(s) * c.Hkv + h) * p.budget;
  const int steps = (m + step - 1) / step;
  const int my_g0 = tid / c.group * c.group;  // first row of this thread's group in a window
  const bool by_shuffle = c.group <= 32 && (c.group & (c.group - 1)) == 0;  // a group lies in one warp
  auto step_barrier = [&]() {
    if (cs > 1) cluster.sync(); else __syncthreads();
  };

  auto position = [&](int w) {  // source position of this thread's row in step w
    const int j = first + w * step + tid;
    return tid < win && w < steps && j < m ? kept[j] : -1;
  };
  // page (-1: none) and row in it of a position
  const int32_t* const table = c.block_tables + s * c.sbt[0];
  const int num_blocks = static_cast<int>(c.num_blocks), max_rows = static_cast<int>(c.max_rows);
  auto page_of = [&](int i, int& row) {
    row = 0;
    if (i < 0 || i >= max_rows) return -1;
    const uint32_t lp = c.by_P(i);
    row = i - static_cast<int>(lp) * c.P;
    const int page = table[lp * c.sbt[1]];
    return page < num_blocks ? page : -1;
  };
  uint8_t* const codes = pl.code + h * pl.sc[1];
  float* const scales = pl.scale + h * pl.ss[1];
  auto place = [&](int page, int row, float*& sc) {  // row and scale addresses
    sc = page < 0 ? nullptr : scales + page * pl.ss[0] + c.by_group(row) * pl.ss[2];
    return page < 0 ? nullptr : codes + page * pl.sc[0] + row * pl.sc[2];
  };
  auto fetch = [&](int w) {  // the rows of step w, whose addresses are in src[w & 1]
    const int rows = max(0, min(win, m - (first + w * step)));
    uint8_t* to = stage + static_cast<size_t>(w & flip) * win * D;
    const uint8_t** from = src + (w & 1) * win;
    if (VEC == 16 && 256 % pieces == 0) {
      const int d = (tid % pieces) * 16;
#pragma unroll 4
      for (int r = tid / pieces; r < rows; r += 256 / pieces) {
        const uint8_t* x = from[r];
        cp_async_16(to + r * D + d, x ? x + d : pl.code, x != nullptr);
      }
    } else {
      for (int e = tid; e < rows * pieces; e += 256) {
        const int r = e / pieces, d = (e - r * pieces) * VEC;
        const uint8_t* x = from[r];
        if (VEC == 16) cp_async_16(to + r * D + d, x ? x + d : pl.code, x != nullptr);
        else to[r * D + d] = x ? x[d * pl.sc[3]] : 0;
      }
    }
  };

  float *sc0, *sc1;
  int i1 = position(1), i2 = position(2), row;
  {
    const int page = page_of(position(0), row);
    uint8_t* x = place(page, row, sc0);
    if (tid < win) src[tid] = x;
  }
  float v0 = sc0 ? *sc0 : 0.f;
  __syncthreads();
  fetch(0);
  {
    const int page = page_of(i1, row);
    uint8_t* x = place(page, row, sc1);
    if (tid < win) src[win + tid] = x;
  }
  cp_async_wait_all();
  step_barrier();
  for (int w = 0; w < steps; ++w) {
    const int j0 = first + w * step, rows = max(0, min(win, m - j0));
    // loads for the steps ahead
    const float v1 = sc1 ? *sc1 : 0.f;
    if (flip && w + 1 < steps) fetch(w + 1);
    int row2, drow;
    const int page2 = page_of(i2, row2);
    const int i3 = position(w + 3);
    const bool mine = tid < rows;
    const int dpage = page_of(mine ? j0 + tid : -1, drow);
    // ---- this step's scales: the largest of each destination group ----
    float v_group = mine ? v0 : 0.f;
    if (by_shuffle) {
      for (int o = 1; o < c.group; o <<= 1) v_group = kv8_scale_max(v_group, __shfl_xor_sync(0xffffffffu, v_group, o));
    } else {
      if (tid < win) was[tid] = v_group;
      __syncthreads();
    }
    if (mine) {
      float big = v_group;
      if (!by_shuffle) {
        big = 0.f;
        for (int r = my_g0; r < min(rows, my_g0 + c.group); ++r) big = kv8_scale_max(big, was[r]);
      }
      float* sc;
      uint8_t* y = place(dpage, drow, sc);
      dst[tid] = {y, v0 < big ? v0 / big : 1.f};
      if (tid == my_g0 && sc) *sc = big;
    }
    __syncthreads();
    // ---- write this step's rows ----
    const uint8_t* from = stage + static_cast<size_t>(w & flip) * win * D;
    auto store16 = [&](int r, int d) {
      uint8_t* y = dst[r].row;
      const float f = dst[r].ratio;
      uint4 q = *reinterpret_cast<const uint4*>(from + r * D + d);
      if (f < 1.f) {
        q.x = kv8_rescale4<CODE>(q.x, f);
        q.y = kv8_rescale4<CODE>(q.y, f);
        q.z = kv8_rescale4<CODE>(q.z, f);
        q.w = kv8_rescale4<CODE>(q.w, f);
      }
      if (y) *reinterpret_cast<uint4*>(y + d) = q;
    };
    if (VEC == 16 && 256 % pieces == 0) {
      const int d = (tid % pieces) * 16;
#pragma unroll 2
      for (int r = tid / pieces; r < rows; r += 256 / pieces) store16(r, d);
    } else {
      for (int e = tid; e < rows * pieces; e += 256) {
        const int r = e / pieces, d = (e - r * pieces) * VEC;
        if (VEC == 16) {
          store16(r, d);
        } else if (dst[r].row) {
          uint8_t q = from[r * D + d];
          if (dst[r].ratio < 1.f) q = Kv8<CODE>::enc(Kv8<CODE>::dec(q) * dst[r].ratio);
          dst[r].row[d * pl.sc[3]] = q;
        }
      }
    }
    if (!flip && w + 1 < steps) {  // one stage: the next step's rows once this one's are out of it
      __syncthreads();
      fetch(w + 1);
    }
    // ---- addresses two steps ahead (their slot's last reader was the fetch of step w) ----
    v0 = v1;
    {
      uint8_t* x = place(page2, row2, sc1);
      if (tid < win) src[(w & 1) * win + tid] = x;
    }
    i2 = i3;
    cp_async_wait_all();
    step_barrier();
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

// Whether clusters of 16 CTAs of this kernel can run (more than eight is not
// portable: it has to be allowed, and a GPC has to have the room).  Asked once per
// device, kernel and shared-memory size.
static bool cluster16_ok(const void* func, int threads, size_t smem) {
  static std::mutex mu;
  static std::map<std::tuple<const void*, int, size_t>, bool> known;
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lock(mu);
  const auto key = std::make_tuple(func, dev, smem);
  const auto it = known.find(key);
  if (it != known.end()) return it->second;
  int n = 0;
  if (cudaFuncSetAttribute(func, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(16);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 16;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, func, &cfg) != cudaSuccess) n = 0;
  }
  if (n == 0) cudaGetLastError();  // not an error of the caller's
  known[key] = n > 0;
  return n > 0;
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
  // ---- move: windows of about 32 KB of rows, a multiple of the group; two of them in
  // shared memory, one where a wide group leaves no room (at most 256 x 640 codes) ----
  int64_t win = 32768 / c.D / c.group * c.group;
  if (win < c.group) win = c.group;
  if (win > 256) win = 256 / c.group * c.group;
  p.window = static_cast<int>(win);
  auto smem_of = [&](int64_t stages) { return (stages * win * c.D + 15) / 16 * 16 + 2 * win * 8 + win * 16 + win * 4; };
  p.stages = smem_of(2) <= 200 * 1024 ? 2 : 1;
  const int smem = static_cast<int>(smem_of(p.stages));
  bool vec = c.D % 16 == 0;
  for (const Kv8Plane& pl : c.plane)
    vec = vec && pl.sc[3] == 1 && (reinterpret_cast<uintptr_t>(pl.code) & 15) == 0 && ((pl.sc[0] | pl.sc[1] | pl.sc[2]) & 15) == 0;
  void (*move)(const Kv8EvictParams) = nullptr;
  TAK_BY_CODE(code_type, move = vec ? kv8_evict_move_kernel<CODE, 16> : kv8_evict_move_kernel<CODE, 1>);
  // (whatever can be refused is refused here: the selection already changes `weights`)
  if (const int r = ensure_smem_attr(reinterpret_cast<const void*>(move), smem)) return r;
  // a cluster per (sequence, head, K or V), of several CTAs where there are fewer
  // of them than fill the SMs
  const int64_t units = 2 * static_cast<int64_t>(c.Hkv) * c.num_seqs;
  int move_cs = 1;
  while (move_cs < 16 && units * move_cs < num_sms() && move_cs * win < budget) move_cs *= 2;
  if (move_cs == 16 && !cluster16_ok(reinterpret_cast<const void*>(move), 256, static_cast<size_t>(smem))) move_cs = 8;

  // ---- selection: in registers up to 8 CTAs x 1024 threads x 16 weights ----
  const int64_t rows = width < c.max_rows ? width : c.max_rows;
  const int64_t sel = kSelThreads;
  note_kernel("kv8_evict");
  if (rows <= 16 * 8 * sel) {
    // eight weights a thread let two CTAs fit an SM; past 8 CTAs of that, sixteen
    // (8 heads of 100000 weights: half the time of eight a thread in clusters of 16)
    const int kpt = rows <= 4 * sel ? 4 : rows <= 8 * 8 * sel ? 8 : 16;
    int cs = 1;
    while (rows > kpt * sel * cs) cs *= 2;
    const dim3 grid(c.Hkv * cs, c.num_seqs);
    int r;
    if (kpt == 4) r = launch_cluster(kv8_evict_select_reg_kernel<4>, grid, kSelThreads, 0, cs, false, st, p);
    else if (kpt == 8) r = launch_cluster(kv8_evict_select_reg_kernel<8>, grid, kSelThreads, 0, cs, false, st, p);
    else r = launch_cluster(kv8_evict_select_reg_kernel<16>, grid, kSelThreads, 0, cs, false, st, p);
    if (r) return r;
  } else {
    kv8_evict_select_kernel<<<dim3(c.Hkv, c.num_seqs), kSelThreads, 0, st>>>(p);
  }
  return launch_cluster(move, dim3(c.Hkv * move_cs, c.num_seqs, 2), 256, static_cast<size_t>(smem), move_cs, true, st, p);
}

}  // namespace tak
