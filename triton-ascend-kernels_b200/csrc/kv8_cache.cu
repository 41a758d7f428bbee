// Writing rows into the 8-bit KV cache and reading them back.
//
// Write: rows of sequence s go to positions [start_s, start_s + n_s).  One CTA
// per (sequence, group of rows, head, K or V): the largest magnitude of the
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
__device__ __forceinline__ int64_t kv8_item_base(const Kv8WriteParams& p, int s) {
  return (p.cu ? p.cu[s] : s) / p.c.group + 2 * static_cast<int64_t>(s);
}

template <typename T, int CODE>
__global__ void __launch_bounds__(128) kv8_write_kernel(const Kv8WriteParams p) {
  const Kv8View& c = p.c;
  int lo = 0, hi = c.num_seqs - 1;
  const int64_t item = blockIdx.x;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (kv8_item_base(p, mid) <= item) lo = mid; else hi = mid - 1;
  }
  const int s = lo, h = blockIdx.y;
  const int64_t tok0 = p.cu ? p.cu[s] : s;
  const int64_t n = p.cu ? p.cu[s + 1] - tok0 : 1;
  const int64_t start = p.start_lens[s];
  const int64_t first = (start / c.group + (item - kv8_item_base(p, s))) * c.group;  // the group's first position
  if (n <= 0 || start < 0 || first >= start + n) return;
  const int64_t page = kv8_page(c, s, first);
  if (page < 0) return;
  const int64_t r0 = max(start, first), r1 = min(start + n, first + c.group);
  const int in_page = static_cast<int>(first % c.P);
  const Kv8Plane& pl = c.plane[blockIdx.z];
  const T* x = static_cast<const T*>(p.x[blockIdx.z]) + (tok0 + (r0 - start)) * p.sx[blockIdx.z][0] +
               h * p.sx[blockIdx.z][1];
  const int64_t st = p.sx[blockIdx.z][0], sd = p.sx[blockIdx.z][2];
  const int held = static_cast<int>(r0 - first), fresh = static_cast<int>(r1 - r0), D = c.D;

  uint32_t amax = 0;
  for (int e = threadIdx.x; e < fresh * D; e += 128)
    amax = max(amax, abs_bits(Elem<T>::to_f(x[(e / D) * st + (e % D) * sd])));
  __shared__ uint32_t red[4];
  amax = __reduce_max_sync(0xffffffffu, amax);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
  __syncthreads();
  amax = max(max(red[0], red[1]), max(red[2], red[3]));
  float* sp = kv8_scale(pl, page, h, in_page / c.group);
  const float was = *sp, want = kv8_scale_of<CODE>(amax);
  const float now = held > 0 ? kv8_scale_max(was, want) : want;
  __syncthreads();  // every thread has read the old scale
  if (threadIdx.x == 0) *sp = now;
  if (held > 0 && was < now) {
    const float ratio = was / now;
    for (int e = threadIdx.x; e < held * D; e += 128) {
      uint8_t* q = kv8_row(pl, page, h, in_page + e / D) + (e % D) * pl.sc[3];
      *q = Kv8<CODE>::enc(Kv8<CODE>::dec(*q) * ratio);
    }
  }
  const float inv = now > 0.f ? 1.0f / now : 0.f;  // 0 for a NaN scale too: its codes are 0
  for (int e = threadIdx.x; e < fresh * D; e += 128) {
    const float v = Elem<T>::to_f(x[(e / D) * st + (e % D) * sd]) * inv;
    kv8_row(pl, page, h, in_page + held + e / D)[(e % D) * pl.sc[3]] = inv > 0.f ? Kv8<CODE>::enc(v) : 0;
  }
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
  const dim3 grid(static_cast<unsigned>(total / c.group + 2 * static_cast<int64_t>(c.num_seqs)), c.Hkv, 2);
  note_kernel("kv8_write");
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

template <typename T, int CODE>
__global__ void __launch_bounds__(128) kv8_read_kernel(const Kv8ReadParams p) {
  const Kv8View& c = p.c;
  const int t = blockIdx.x;
  if (c.num_seqs == 0) return;
  const int s = find_slot_seq(p.cu, c.num_seqs, t);
  const bool in_seq = t >= p.cu[s] && t < p.cu[s + 1];
  const int64_t pos = in_seq ? t - p.cu[s] + (p.start_lens ? p.start_lens[s] : 0) : -1;
  const int64_t page = kv8_page(c, s, pos);
  const int row = page >= 0 ? static_cast<int>(pos % c.P) : 0;
  for (int e = threadIdx.x; e < 2 * c.Hkv * c.D; e += 128) {
    const int w = e / (c.Hkv * c.D), h = e / c.D % c.Hkv, d = e % c.D;
    const Kv8Plane& pl = c.plane[w];
    float v = 0.f;
    if (page >= 0)
      v = Kv8<CODE>::dec(kv8_row(pl, page, h, row)[d * pl.sc[3]]) * *kv8_scale(pl, page, h, row / c.group);
    static_cast<T*>(p.y[w])[t * p.sy[w][0] + h * p.sy[w][1] + d * p.sy[w][2]] = Elem<T>::from_f(v);
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
  note_kernel("kv8_read");
  TAK_BY_DTYPE(dtype, TAK_BY_CODE(code_type, kv8_read_kernel<T, CODE><<<static_cast<unsigned>(total), 128, 0, st>>>(p)));
  return 0;
}

}  // namespace tak
