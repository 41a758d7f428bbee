// Writing rows into the 8-bit KV cache and reading them back.
//
// Write: rows of sequence s go to positions [start_s, start_s + n_s).  One work
// item per (sequence, group of rows, head, K or V): the largest magnitude of the
// group's new rows gives a scale; where the group already holds rows (its first
// position lies before start_s) the scale is the larger of that and the stored
// one, and rows held under a smaller scale are requantised,
//   code' = round(code * (old scale / new scale)).
// Codes of new rows are round(x * (1 / scale)), to nearest even.
#include "kv8.cuh"

namespace tak {

struct Kv8WriteParams {
  Kv8View c;
  const void* x[2]; int64_t sx[2][3];
  const int32_t* start_lens;
  const int32_t* cu;  // null: one row per sequence
  int64_t total;
};

// Work items of a sequence: group g of its rows [start, start + n).  Sequence s
// owns items [cu[s] / group + 2 s, cu[s + 1] / group + 2 (s + 1)), at least as
// many as the groups that n rows can touch, so the list needs no prefix sums.
// Without cu each sequence has one row and one item.
__device__ __forceinline__ int64_t kv8_item_base(const Kv8WriteParams& p, int s) {
  return p.cu ? p.cu[s] / p.c.group + 2 * static_cast<int64_t>(s) : s;
}

// What an item writes: rows [r0, r0 + fresh) of sequence s, after `held` rows that
// the group has.
struct Kv8WriteItem {
  int s, held, fresh, in_page;
  int64_t page, token;
};
__device__ __forceinline__ bool kv8_write_item(const Kv8WriteParams& p, int64_t item, Kv8WriteItem& w) {
  const Kv8View& c = p.c;
  int lo = 0;
  if (p.cu) {
    // last sequence whose items begin at or before `item`, 32 candidates a round
    // (every lane of the warp looks at the same item)
    for (int span = c.num_seqs; span > 1;) {
      const int step = (span + 31) / 32, s = lo + static_cast<int>(threadIdx.x & 31) * step;
      const unsigned le = __ballot_sync(0xffffffffu, s < c.num_seqs && s < lo + span && kv8_item_base(p, s) <= item);
      const int at = 31 - __clz(le | 1u);
      span = min(step, span - at * step);
      lo += at * step;
    }
  } else {
    lo = static_cast<int>(item);
  }
  const int64_t tok0 = p.cu ? p.cu[lo] : lo;
  const int64_t n = p.cu ? min(static_cast<int64_t>(p.cu[lo + 1]), p.total) - tok0 : 1;
  const int64_t start = p.start_lens[lo];
  if (n <= 0 || tok0 < 0 || start < 0) return false;
  const int64_t first = (static_cast<int64_t>(c.by_group(static_cast<uint32_t>(start))) + (item - kv8_item_base(p, lo))) * c.group;  // the group's first position
  if (first >= start + n) return false;
  w.s = lo;
  w.page = kv8_page(c, lo, first);
  if (w.page < 0) return false;
  const int64_t r0 = max(start, first), r1 = min(start + n, first + c.group);
  w.in_page = static_cast<int>(first - static_cast<int64_t>(c.by_P(static_cast<uint32_t>(first))) * c.P);  // page >= 0: first < 2^31
  w.token = tok0 + (r0 - start);
  w.held = static_cast<int>(r0 - first);
  w.fresh = static_cast<int>(r1 - r0);
  return true;
}

// Eight elements of a row, as loaded (16-bit types: one 16-byte word), and the
// running maximum of magnitudes over such pieces.  The maxima keep NaN.
template <typename T> struct Pair;
template <> struct Pair<__half> { using type = __half2; };
template <> struct Pair<__nv_bfloat16> { using type = __nv_bfloat162; };
template <typename T> struct Eight {
  using P = typename Pair<T>::type;
  uint4 v;
  struct Max {
    uint32_t m = 0;
    __device__ __forceinline__ uint32_t bits() const {
      const float2 f = Elem<T>::unpack2(m);
      return max(abs_bits(f.x), abs_bits(f.y));
    }
  };
  __device__ __forceinline__ void load(const T* x) { v = *reinterpret_cast<const uint4*>(x); }
  __device__ __forceinline__ void into(Max& a) const {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
    P m = *reinterpret_cast<P*>(&a.m);
#pragma unroll
    for (int k = 0; k < 4; ++k) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const P*>(&u[k])));
    a.m = *reinterpret_cast<uint32_t*>(&m);
  }
  __device__ __forceinline__ void get(float* f) const {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 t = Elem<T>::unpack2(u[k]);
      f[2 * k] = t.x;
      f[2 * k + 1] = t.y;
    }
  }
};
template <> struct Eight<float> {
  float4 a, b;
  struct Max {
    uint32_t m = 0;
    __device__ __forceinline__ uint32_t bits() const { return m; }
  };
  __device__ __forceinline__ void load(const float* x) {
    a = *reinterpret_cast<const float4*>(x);
    b = *reinterpret_cast<const float4*>(x + 4);
  }
  __device__ __forceinline__ void into(Max& x) const {
    float f[8];
    get(f);
#pragma unroll
    for (int i = 0; i < 8; ++i) x.m = max(x.m, abs_bits(f[i]));
  }
  __device__ __forceinline__ void get(float* f) const {
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
};

// One item held in registers: TPI threads (one warp, or a CTA of its own), up to
// eight pieces of eight elements each of K and of V, so the rows are read once.
// TPI is the least that holds the group: a warp for 16 rows of 128.
//
// Bound by memory latency and issue slots alike (59 % issue): 34816 rows of 8 heads x
// 128 in 45 to 48 us (214 MB, 4.5 TB/s, 69 % of the measured copy rate).  Pieces at
// fixed pointer steps took a fifth fewer instructions and 3 us more: loads and their
// registers spread out less well.  One row for each of 64 requests takes 3.6 us.
template <typename T, int CODE, int TPI>
__global__ void __launch_bounds__(TPI == 32 ? 128 : TPI) kv8_write_vec_kernel(const Kv8WriteParams p, int64_t items) {
  constexpr int U = 8;
  const Kv8View& c = p.c;
  const int lane = threadIdx.x % TPI;
  // the heads of an item are neighbours: they read the same rows
  uint32_t id = TPI == 32 ? blockIdx.x * 4 + threadIdx.x / 32 : blockIdx.x;  // units < 2^31
  const int h = id % static_cast<uint32_t>(c.Hkv);
  id /= static_cast<uint32_t>(c.Hkv);
  Kv8WriteItem w;
  if (id >= items || !kv8_write_item(p, id, w)) return;
  const int pr = c.D / 8, n = w.fresh * pr;  // pieces of a row, of the item
  // piece k of this thread: row and piece of it (one division where the threads
  // cover whole rows)
  const int lr = lane / pr, lc = lane - lr * pr, step = TPI / pr;
  const bool whole = step * pr == TPI;
  auto place = [&](int k, int& r, int& d) {
    r = whole ? lr + k * step : (lane + k * TPI) / pr;
    d = (whole ? lc : (lane + k * TPI) - r * pr) * 8;
  };
  Eight<T> v[2][U];
  float* sp[2];
  float was[2];
#pragma unroll
  for (int which = 0; which < 2; ++which) {  // K and V in flight together
    const T* x = static_cast<const T*>(p.x[which]) + w.token * p.sx[which][0] + h * p.sx[which][1];
    sp[which] = kv8_scale(c.plane[which], w.page, h, w.in_page / c.group);
    was[which] = *sp[which];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      int r, d;
      place(k, r, d);
      if (lane + k * TPI < n) v[which][k].load(x + r * p.sx[which][0] + d);
    }
  }
  uint32_t amax[2];
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    typename Eight<T>::Max top;
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (lane + k * TPI < n) v[which][k].into(top);
    amax[which] = __reduce_max_sync(0xffffffffu, top.bits());
  }
  if (TPI > 32) {
    __shared__ uint2 red[TPI / 32];
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_uint2(amax[0], amax[1]);
    __syncthreads();  // also: every thread has read the old scales
#pragma unroll
    for (int i = 0; i < TPI / 32; ++i) {
      amax[0] = max(amax[0], red[i].x);
      amax[1] = max(amax[1], red[i].y);
    }
  }
  __syncwarp();
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const Kv8Plane& pl = c.plane[which];
    const float want = kv8_scale_of<CODE>(amax[which]), now = w.held > 0 ? kv8_scale_max(was[which], want) : want;
    if (lane == 0) *sp[which] = now;
    uint8_t* const row0 = kv8_row(pl, w.page, h, w.in_page);
    if (w.held > 0 && was[which] < now) {
      const float ratio = was[which] / now;
      for (int e = lane; e < w.held * pr; e += TPI) {
        uint2* q = reinterpret_cast<uint2*>(row0 + (e / pr) * pl.sc[2] + (e % pr) * 8);
        uint2 t = *q;
        t.x = kv8_rescale4<CODE>(t.x, ratio);
        t.y = kv8_rescale4<CODE>(t.y, ratio);
        *q = t;
      }
    }
    const float inv = now > 0.f ? 1.0f / now : 0.f;
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (lane + k * TPI >= n) continue;
      int r, d;
      place(k, r, d);
      uint2 q = make_uint2(0, 0);
      if (now > 0.f) {  // else (zeros, or a NaN scale) the codes are 0
        float f[8];
        v[which][k].get(f);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = __fmul_rn(f[i], inv);
        q = make_uint2(kv8_enc4<CODE>(f), kv8_enc4<CODE>(f + 4));
      }
      *reinterpret_cast<uint2*>(row0 + (w.held + r) * pl.sc[2] + d) = q;
    }
  }
}

// Any layout and size: one CTA per item, the rows read twice.
template <typename T, int CODE>
__global__ void __launch_bounds__(128) kv8_write_kernel(const Kv8WriteParams p) {
  const Kv8View& c = p.c;
  const int h = blockIdx.y, which = blockIdx.z, D = c.D;
  Kv8WriteItem w;
  if (!kv8_write_item(p, blockIdx.x, w)) return;
  const Kv8Plane& pl = c.plane[which];
  const T* x = static_cast<const T*>(p.x[which]) + w.token * p.sx[which][0] + h * p.sx[which][1];
  const int64_t st = p.sx[which][0], sd = p.sx[which][2];
  uint32_t amax = 0;
  for (int e = threadIdx.x; e < w.fresh * D; e += 128)
    amax = max(amax, abs_bits(Elem<T>::to_f(x[(e / D) * st + (e % D) * sd])));
  __shared__ uint32_t red[4];
  amax = __reduce_max_sync(0xffffffffu, amax);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
  float* sp = kv8_scale(pl, w.page, h, w.in_page / c.group);
  const float was = *sp;
  __syncthreads();  // every thread has read the old scale
  amax = max(max(red[0], red[1]), max(red[2], red[3]));
  const float want = kv8_scale_of<CODE>(amax), now = w.held > 0 ? kv8_scale_max(was, want) : want;
  if (threadIdx.x == 0) *sp = now;
  if (w.held > 0 && was < now) {
    const float ratio = was / now;
    for (int e = threadIdx.x; e < w.held * D; e += 128) {
      uint8_t* q = kv8_row(pl, w.page, h, w.in_page + e / D) + (e % D) * pl.sc[3];
      *q = Kv8<CODE>::enc(Kv8<CODE>::dec(*q) * ratio);
    }
  }
  const float inv = now > 0.f ? 1.0f / now : 0.f;
  for (int e = threadIdx.x; e < w.fresh * D; e += 128) {
    const float v = Elem<T>::to_f(x[(e / D) * st + (e % D) * sd]) * inv;
    kv8_row(pl, w.page, h, w.in_page + w.held + e / D)[(e % D) * pl.sc[3]] = inv > 0.f ? Kv8<CODE>::enc(v) : 0;
  }
}

// rows of codes in whole aligned pieces of n codes
static bool codes_vec_ok(const Kv8View& c, int n) {
  if (c.D % n) return false;
  for (const Kv8Plane& pl : c.plane)
    if (pl.sc[3] != 1 || (reinterpret_cast<uintptr_t>(pl.code) & (n - 1)) || ((pl.sc[0] | pl.sc[1] | pl.sc[2]) & (n - 1))) return false;
  return true;
}
// rows of T in 16-byte pieces
static bool rows_vec_ok(const void* x, const int64_t* st, int size) {
  const int n = 16 / size;
  return st[2] == 1 && (reinterpret_cast<uintptr_t>(x) & 15) == 0 && ((st[0] | st[1]) & (n - 1)) == 0;
}

int kv8_write_launch(const Kv8View& c, int code_type, const void* k, const int64_t* sk, const void* v,
                     const int64_t* sv, const int32_t* start_lens, const int32_t* cu, int64_t total, int dtype,
                     cudaStream_t st) {
  Kv8WriteParams p{};
  p.c = c;
  p.x[0] = k; p.x[1] = v;
  for (int i = 0; i < 3; ++i) { p.sx[0][i] = sk[i]; p.sx[1][i] = sv[i]; }
  p.start_lens = start_lens;
  p.cu = cu;
  p.total = total;
  const int64_t items = cu ? total / c.group + 2 * static_cast<int64_t>(c.num_seqs) : c.num_seqs;
  const int size = dtype == kF32 ? 4 : 2;
  note_kernel("kv8_write");
  const int pieces = c.group * (c.D / 8);  // of eight elements; a thread holds up to eight
  if (codes_vec_ok(c, 8) && rows_vec_ok(k, sk, size) && rows_vec_ok(v, sv, size) && pieces <= 8 * 512 &&
      items * c.Hkv < (int64_t{1} << 31)) {
    const int64_t units = items * c.Hkv;  // K and V together
    const unsigned warps = static_cast<unsigned>((units + 3) / 4), ctas = static_cast<unsigned>(units);
    TAK_BY_DTYPE(dtype, TAK_BY_CODE(code_type, {
      if (pieces <= 8 * 32) kv8_write_vec_kernel<T, CODE, 32><<<warps, 128, 0, st>>>(p, items);
      else if (pieces <= 8 * 128) kv8_write_vec_kernel<T, CODE, 128><<<ctas, 128, 0, st>>>(p, items);
      else kv8_write_vec_kernel<T, CODE, 512><<<ctas, 512, 0, st>>>(p, items);
    }));
    return 0;
  }
  const dim3 grid(static_cast<unsigned>(items), c.Hkv, 2);
  TAK_BY_DTYPE(dtype, TAK_BY_CODE(code_type, kv8_write_kernel<T, CODE><<<grid, 128, 0, st>>>(p)));
  return 0;
}

struct Kv8ReadParams {
  Kv8View c;
  void* y[2]; int64_t sy[2][3];
  const int32_t* start_lens;  // may be null: rows from position 0
  const int32_t* cu;
  int64_t total;
};

// A warp reads TB (at most 32) consecutive tokens: lane i looks up token i's page,
// then the warp walks the tokens with each lane on its piece of a head, K and V
// together, the next token's codes in flight while these are converted.  VEC codes a
// piece (16: one load, 32 bytes of 16-bit values or 64 of fp32 out).
//
// Bound by memory, two thirds of it writes: 69632 rows of 8 heads x 128 (e4m3 to
// fp16) in 81 us, 5.27 TB/s, 80 % of the measured copy rate.  CTAs that looked 16 to
// 32 tokens up behind a barrier took 88 to 95 us.
template <typename T, int VEC> struct Kv8Piece;
template <typename T> struct Kv8Piece<T, 16> {
  uint4 q;
  __device__ __forceinline__ void load(const uint8_t* x) { q = *reinterpret_cast<const uint4*>(x); }
  template <int CODE> __device__ __forceinline__ void store(T* out, float sc) const {
    const uint32_t u[4] = {q.x, q.y, q.z, q.w};
    float f[16];
#pragma unroll
    for (int k = 0; k < 4; ++k) kv8_dec4<CODE>(u[k], f + 4 * k);
#pragma unroll
    for (int k = 0; k < 16; ++k) f[k] *= sc;
    if constexpr (sizeof(T) == 2) {
      uint32_t o[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) o[k] = Elem<T>::pack2(f[2 * k], f[2 * k + 1]);
      reinterpret_cast<uint4*>(out)[0] = make_uint4(o[0], o[1], o[2], o[3]);
      reinterpret_cast<uint4*>(out)[1] = make_uint4(o[4], o[5], o[6], o[7]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        reinterpret_cast<float4*>(out)[k] = make_float4(f[4 * k], f[4 * k + 1], f[4 * k + 2], f[4 * k + 3]);
    }
  }
};
template <typename T> struct Kv8Piece<T, 1> {
  uint8_t q;
  __device__ __forceinline__ void load(const uint8_t* x) { q = *x; }
  template <int CODE> __device__ __forceinline__ void store(T* out, float sc) const {
    *out = Elem<T>::from_f(Kv8<CODE>::dec(q) * sc);
  }
};

template <typename T, int CODE, int VEC>
__global__ void __launch_bounds__(256, 4) kv8_read_kernel(const __grid_constant__ Kv8ReadParams p, int TB) {
  const Kv8View& c = p.c;
  const int lane = threadIdx.x & 31;
  const int64_t t0 = (static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5)) * TB;
  const int tn = static_cast<int>(min(static_cast<int64_t>(TB), p.total - t0));
  if (tn <= 0) return;
  int my_page = -1, my_row = 0;
  if (lane < tn) {
    const int64_t t = t0 + lane;
    const int s = find_slot_seq(p.cu, c.num_seqs, t);
    const int lo = p.cu[s];
    if (t >= lo && t < p.cu[s + 1]) {
      const int64_t pos = t - lo + (p.start_lens ? p.start_lens[s] : 0);
      my_page = static_cast<int>(kv8_page(c, s, pos));  // num_blocks < 2^31
      if (my_page >= 0) my_row = static_cast<int>(pos - static_cast<int64_t>(c.by_P(static_cast<uint32_t>(pos))) * c.P);
    }
  }
  const int pr = c.D / VEC, per_tok = c.Hkv * pr;
  for (int e = lane; e < (per_tok + 31) / 32 * 32; e += 32) {
    const bool live = e < per_tok;
    const int h = live ? e / pr : 0, d = live ? (e - h * pr) * VEC : 0;
    const uint8_t* code[2];
    const float* scale[2];
    T* out[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      code[w] = c.plane[w].code + h * c.plane[w].sc[1] + d * (VEC > 1 ? 1 : c.plane[w].sc[3]);
      scale[w] = c.plane[w].scale + h * c.plane[w].ss[1];
      out[w] = static_cast<T*>(p.y[w]) + t0 * p.sy[w][0] + h * p.sy[w][1] + d * (VEC > 1 ? 1 : p.sy[w][2]);
    }
    Kv8Piece<T, VEC> next[2];
    float next_sc[2];
    auto load = [&](int i) {
      const int page = __shfl_sync(0xffffffffu, my_page, i), row = __shfl_sync(0xffffffffu, my_row, i);
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        next[w] = {};
        next_sc[w] = 0.f;
        if (page >= 0 && live) {
          next[w].load(code[w] + page * c.plane[w].sc[0] + row * c.plane[w].sc[2]);
          next_sc[w] = scale[w][page * c.plane[w].ss[0] + static_cast<int64_t>(c.by_group(row)) * c.plane[w].ss[2]];
        }
      }
    };
    load(0);
    for (int i = 0; i < tn; ++i) {
      Kv8Piece<T, VEC> now[2];
      float sc[2];
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        now[w] = next[w];
        sc[w] = next_sc[w];
      }
      if (i + 1 < tn) load(i + 1);
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        if (live) now[w].template store<CODE>(out[w], sc[w]);
        out[w] += p.sy[w][0];
      }
    }
  }
}

int kv8_read_launch(const Kv8View& c, int code_type, const int32_t* cu, const int32_t* start_lens, int64_t total,
                    void* k, const int64_t* sk, void* v, const int64_t* sv, int dtype, cudaStream_t st) {
  Kv8ReadParams p{};
  p.c = c;
  p.y[0] = k; p.y[1] = v;
  for (int i = 0; i < 3; ++i) { p.sy[0][i] = sk[i]; p.sy[1][i] = sv[i]; }
  p.start_lens = start_lens;
  p.cu = cu;
  p.total = total;
  const int size = dtype == kF32 ? 4 : 2;
  const bool vec = codes_vec_ok(c, 16) && rows_vec_ok(k, sk, size) && rows_vec_ok(v, sv, size);
  // tokens of a warp (their pages are looked up in one go): fewer where the GPU
  // would not be filled
  const int64_t warps = 32 * static_cast<int64_t>(num_sms());
  const int tb = total >= 16 * 2 * warps ? 16 : total >= 4 * warps ? 8 : total >= warps ? 2 : 1;
  const unsigned grid = static_cast<unsigned>((total + 8 * tb - 1) / (8 * tb));
  note_kernel("kv8_read");
  TAK_BY_DTYPE(dtype, TAK_BY_CODE(code_type, {
    if (vec) kv8_read_kernel<T, CODE, 16><<<grid, 256, 0, st>>>(p, tb);
    else kv8_read_kernel<T, CODE, 1><<<grid, 256, 0, st>>>(p, tb);
  }));
  return 0;
}

}  // namespace tak
