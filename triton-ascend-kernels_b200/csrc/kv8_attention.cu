// Attention over the 8-bit KV cache: split over the keys, one pass.
//
// Mathematics.  With codes Kc, Vc and a scale for each group of rows, a row's
// score against key j is s_j = scale * ks_g (q . Kc_j) and its output
// sum_j p_j vs_g Vc_j.  Both scales are constant over a tile of 16 keys (groups
// are multiples of 16), so K's scale multiplies a tile's scores and V's goes
// into the exponent: with lv = log2(vs),
//   P_j = 2^(s_j + lv - M),  O = sum_j P_j Vc_j,  l = sum_j 2^(s_j - M),  out = O / l,
// where M is the running maximum of s_j + lv, and l's terms are P_j / vs unless V's
// scales lie far apart (kFar).  P stays within fp16 whatever the scales are (a small V
// under a large weight and a large V under a small weight are compared by their
// product), and codes are exact in fp16, so both products run on fp16 tensor cores with
// fp32 sums; q is brought to fp16 by a power of two per row, which is exact for
// elements within 2^-22 of the row's largest.  P's rounding to fp16 (2^-11 of each
// weight) is what the 16-bit product costs: nothing to be seen in a bf16 output (error
// 1.7e-3 of its size with or without), but it takes fp16 outputs from 2.1e-4 to as
// much as 2.8e-4 (131071 keys).
//
// Work split.  A (sequence, KV head, chunk of query rows) is an item; an item is
// cut into chunks of CH keys.  The chunks of all items, in order, are dealt out
// evenly: CTA c of N takes chunks [U c / N, U (c + 1) / N), so ragged contexts
// cost no idle SM and the host needs no lengths.  An item inside one CTA is
// finished there; the parts of a cut one go to the workspace (each CTA has at
// most two) and a second grid joins them in order.
//
// A CTA: one producer warp streams chunks through a ring of TMA loads (K and V
// codes, page ids from the block table) with the tiles' scales beside them; NW
// warps consume, in one of two ways: up to eight query rows (Kv8Few), or 16 and 32
// (Kv8Many; more rows are chunks of 32 that share the L2's copy of the cache).
#include <cstdio>

#include "kv8.cuh"

namespace tak {

int kv8_attention_generic_launch(const Kv8View& c, const Kv8AttnArgs& a, cudaStream_t st);

struct Kv8TcParams {
  Kv8View c;
  const void* q; int64_t sq[4];
  const int32_t* context_lens;
  void* out; int64_t so[4];
  float* lse;
  int bf16;          // q and out are bf16 (else fp16)
  int q_vec;         // four consecutive elements of q are one aligned 8-byte word
  int H, Lq, G, rows, chunks;  // rows = G * Lq query rows per KV head, in `chunks` chunks
  int box_rows;      // rows of one TMA box: the largest power of two dividing block_size, at most CH
  float scale;       // softmax scale * log2(e); with a cap: softmax scale
  float cap2, inv_cap;  // softcap * log2(e), 1 / softcap; 0: no cap
  // workspace
  int64_t* places;   // U, the length of the work list
  int4* bound;       // [N] first chunk of each CTA: {sequence, item of it, chunk of the item, chunks of the item}
  float* part_o;     // [N][2][RT][DP]
  float* part_ml;    // [N][2][RT][2]
  float* lse2;       // [B, Hkv, rows] (weights only)
  float* scores;     // [B, Hkv, chunks, RT, score_ld] (weights only)
  int64_t score_ld;
};

// P is held times 2^kPBias: with the running maximum allowed to lag by kLag it
// reaches 2^15 (fp16 ends at 2^16), and weights down to 2^-27 of the largest
// keep fp16's full precision.  Smaller ones, down to 2^-61, are summed apart while a
// row has fewer than kFew larger ones; below that a weight adds nothing to O (it
// still does to l).  l holds the sum of 2^(s - M - kLBias), formed as P / vs while
// every V scale of the item lies within 2^kFar of 1.  From the first tile of another
// scale on (0 among them) P may underflow where the score does not, or 1 / vs leave
// fp32's normal numbers, so l is summed from the scores themselves (kv8_add_term).  With
// M - s between -109 and 121 for the heaviest key, it stays in fp32 (at the upper end
// with 18 bits) for up to 2^26 keys.
constexpr float kPBias = 13.f;
constexpr float kLag = 2.f;
constexpr float kLBias = 10.f;
constexpr float kLBiasInv = 1.1920928955078125e-7f;  // 2^-(kPBias + kLBias)
constexpr float kNoMax = -3e38f;             // maximum of a row that has seen no key: finite, so that no difference is inf - inf
constexpr float kHalfMin = 6.103515625e-5f;  // 2^-14: fp16's smallest normal number
constexpr int kFew = 8;
constexpr float kFar = 48.f;
// The smallest scale that a write makes is 2^-100 / 448 (e4m3); one of kMinVs or less
// is 0.  Its keys count in the maximum as if it were kMinVs, for l's sake, and have P = 0.
constexpr float kMinVs = 1.5407439555097887e-33f;  // 2^-109
constexpr float kMinLv = kPBias - 109.f;

// DP: head dim rounded up to 64, 128 or 256.
template <int DP> struct Kv8Base {
  static constexpr int NW = DP >= 256 ? 8 : 4;          // consumer warps
  static constexpr int CH = 128;                        // keys of a chunk
  static constexpr int TP = CH / 16 / NW;               // key tiles of a warp's step (two: independent MMA chains)
  static constexpr int NT = CH / 16;                    // key tiles of a chunk
  static constexpr int CB = DP >= 256 ? 2 : 1;          // column blocks of a row
  static constexpr int ROWB = DP >= 128 ? 128 : 64;     // bytes of a row in a column block
  static constexpr int PLANE = CH * DP;                 // bytes of K (or V) in a stage
  static constexpr int STAGE = 2 * PLANE;
  static constexpr int NS = DP == 64 ? 4 : 2;
  static constexpr int THREADS = (NW + 1) * 32;
  static constexpr int META_OFF = NS * STAGE;           // [NS][3][NT] floats: ks, log2 vs + kPBias, 2^-23 / vs or 0
  static constexpr int BAR_OFF = META_OFF + NS * 3 * NT * 4;
  static constexpr int OWN_OFF = BAR_OFF + 2 * NS * 8;  // the kernel's own shared memory
};
// Up to eight query rows: every warp holds all of O for its key tiles, and the
// warps join at the end of an item.
template <int DP> struct Kv8Few : Kv8Base<DP> {
  using B = Kv8Base<DP>;
  static constexpr int RT = 8;
  static constexpr int CTAS = DP >= 256 ? 1 : 3;        // per SM
  static constexpr int DH = 64;                         // columns joined at a time
  static constexpr int OLD = DH + 8;                    // row stride of the joining buffer (bank spread)
  static constexpr int OBUF_OFF = B::OWN_OFF;           // [NW][8][OLD] floats
  static constexpr int ML_OFF = OBUF_OFF + B::NW * 8 * OLD * 4;  // [NW][8][2]
  static constexpr int SMEM = ML_OFF + B::NW * 8 * 2 * 4 + 1024;
  static_assert((SMEM + 1024) * CTAS <= 228 * 1024, "shared memory");
};
// 16 or 32 query rows (8 NR): a warp scores its key tiles for all rows, the weights
// go to the other warps through shared memory, and each warp sums its share of the
// columns over all keys of the chunk, so that a code is converted once per CTA.
template <int DP, int NR> struct Kv8Many : Kv8Base<DP> {
  using B = Kv8Base<DP>;
  static constexpr int RT = 8 * NR;
  static constexpr int CTAS = DP >= 256 ? 1 : 2;        // per SM
  static constexpr int CW = DP / B::NW;                 // columns of a warp
  static constexpr int MB = CW / 16;
  static constexpr int Q_OFF = (B::OWN_OFF + 15) / 16 * 16;        // [DP / 16][NR][32 lanes] uint2: Q fragments
  static constexpr int P_OFF = Q_OFF + DP / 16 * NR * 256;         // [2][NT][NR][32 lanes] uint2: P fragments, and those apart
  static constexpr int FAC_OFF = P_OFF + 2 * B::NT * NR * 256;     // [RT] floats
  static constexpr int MAX_OFF = FAC_OFF + RT * 4;                 // [NW][RT] floats
  static constexpr int FLAG_OFF = MAX_OFF + B::NW * RT * 4;        // [2][NW] ints
  static constexpr int SMEM = FLAG_OFF + 2 * B::NW * 4 + 1024;
  static_assert((SMEM + 1024) * CTAS <= 228 * 1024, "shared memory");
};

// byte offset of 16-byte piece `c` of row `r` in a column block
template <int DP> __device__ __forceinline__ uint32_t kv8_sw(uint32_t r, uint32_t c) {
  if (DP >= 128) return r * 128u + ((c ^ (r & 7u)) << 4);
  return r * 64u + ((c ^ ((r >> 1) & 3u)) << 4);
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t d;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(sel));
  return d;
}
__device__ __forceinline__ uint32_t hsub2_1152(uint32_t x) {
  const __half2 k = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
  __half2 h = __hsub2(*reinterpret_cast<__half2*>(&x), k);
  return *reinterpret_cast<uint32_t*>(&h);
}
// transpose of an 8 x 8 matrix of 16-bit elements held as the MMA fragments are
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
}
// Four codes to two fp16 pairs.  int8: the byte with its sign bit flipped goes
// into the mantissa of 1024 (fp16 0x6400, where an ulp is 1): 1024 + 128 + x,
// less 1152.  PAIR = 0 pairs bytes (0,1) (2,3), PAIR = 1 bytes (0,2) (1,3).
template <int CODE, int PAIR>
__device__ __forceinline__ void codes_to_half(uint32_t r, uint32_t& lo, uint32_t& hi) {
  if (CODE == kI8) {
    const uint32_t x = r ^ 0x80808080u;
    lo = hsub2_1152(prmt(x, 0x64646464u, PAIR ? 0x4240 : 0x4140));
    hi = hsub2_1152(prmt(x, 0x64646464u, PAIR ? 0x4341 : 0x4342));
  } else {
    const uint32_t x = PAIR ? prmt(r, 0, 0x3120) : r;
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(x));
  }
}

// Four scores z to cap * tanh(z / cap), in base-2 units (cap2 = cap * log2(e)).
// Below |z / cap| = 0.6, where ordinary scores lie, tanh is its odd polynomial
// (fitted to 8.1e-8 relative); past it, 1 - 2 / (1 + e^(2 z / cap)), whose absolute
// error of 1e-7 is small there.  A warp leaves the second out when it needs it for
// no score.
__device__ __forceinline__ void kv8_cap(float (&x)[4], float inv_cap, float cap2) {
  float t[4];
  bool far = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float h = x[e] * inv_cap, u = h * h;
    float r = fmaf(-0.006276387721300125f, u, 0.021116213873028755f);
    r = fmaf(r, u, -0.053875137120485306f);
    r = fmaf(r, u, 0.13332924246788025f);
    r = fmaf(r, u, -0.3333333134651184f);
    t[e] = fmaf(h * u, r, h);
    far |= fabsf(h) > 0.6f;
  }
  if (__any_sync(0xffffffffu, far)) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float h = x[e] * inv_cap;
      const float big = 1.f - __fdividef(2.f, 1.f + fast_exp2(h * (2.f * kLog2e)));
      t[e] = fabsf(h) > 0.6f ? big : t[e];
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = t[e] * cap2;
}

// l + 2^(x - kLBias), and l + v 2^d with h = 2^(d / 2): by two factors, as the product
// may be subnormal (ex2 ends at 2^-126) and v 2^d be normal where 2^d is not
__device__ __forceinline__ float kv8_add_term(float l, float x) {
  const float h = fast_exp2(fmaf(0.5f, x, -0.5f * kLBias));
  return fmaf(h, h, l);
}
__device__ __forceinline__ float kv8_add_down(float l, float v, float h) { return fmaf(v * h, h, l); }
// out = o * pre * inv: 2^-(kPBias + kLBias) / l, in two factors where one would be subnormal
__device__ __forceinline__ float2 kv8_over(float l) {
  const bool large = l > 18446744073709551616.f;  // 2^64
  const float inv = l != 0.f ? (large ? kLBiasInv * 18446744073709551616.f : kLBiasInv) / l : 0.f;
  return make_float2(large ? 5.42101086242752217e-20f : 1.f, inv);
}

__device__ __forceinline__ int kv8_ctx(const Kv8TcParams& p, int s) {
  const int64_t n = min(static_cast<int64_t>(p.context_lens[s]), p.c.max_rows);
  return n > 0 ? static_cast<int>(n) : 0;
}

// query row `row` (token row / G, head kvh * G + row % G) of a KV head
__device__ __forceinline__ const uint16_t* kv8_q_row(const Kv8TcParams& p, int s, int kvh, int row) {
  const int i = row / p.G;
  return static_cast<const uint16_t*>(p.q) + s * p.sq[0] + i * p.sq[1] + (kvh * p.G + row - i * p.G) * p.sq[2];
}

// Positions in the work list: an item of n chunks takes n + kItemCost places, the
// last kItemCost of them empty.  They stand for what an item costs besides its
// chunks (query rows, joining the warps, the output), so that CTAs with many short
// items get fewer chunks.  (64 x <= 8192 keys, 4 rows a head: 98 to 101 us from 1 to
// 4; 32 rows: 244 us without, 221, 202, 190, 190 us from 1 to 4.)
constexpr int kItemCost = 3;
template <int CH> __device__ __forceinline__ int64_t kv8_places(int ctx) {
  return ctx > 0 ? (ctx + CH - 1) / CH + kItemCost : 0;
}

// Walks a CTA's chunks in order: item `r` of sequence `s`, chunk `j` of `n`, at
// place `at`.
template <int CH> struct Kv8Walk {
  int64_t at;
  int s, r, j, n, ctx;
  __device__ __forceinline__ void load(const Kv8TcParams& p) {
    ctx = kv8_ctx(p, s);
    n = (ctx + CH - 1) / CH;
  }
  __device__ __forceinline__ void next_item(const Kv8TcParams& p, int items) {
    at += n - j + kItemCost;
    j = 0;
    if (++r < items) return;
    r = 0;
    do {
      if (++s >= p.c.num_seqs) return;
      load(p);
    } while (n == 0);
  }
  __device__ __forceinline__ void next(const Kv8TcParams& p, int items) {
    if (j + 1 < n) {
      ++j;
      ++at;
    } else {
      next_item(p, items);
    }
  }
  __device__ __forceinline__ bool live(const Kv8TcParams& p, int64_t end) const { return at < end && s < p.c.num_seqs; }
};

// Start of both kernels: barriers, the CTA's share [w0.at, u1) of the work list,
// zeros for sequences without a key.  False: the CTA has no chunk.
template <class C>
__device__ __forceinline__ bool kv8_begin(const Kv8TcParams& p, uint64_t* full, uint64_t* empty, Kv8Walk<C::CH>& w0, int64_t& u1) {
  constexpr int NW = C::NW, CH = C::CH, NS = C::NS, THREADS = C::THREADS;
  __shared__ int64_t sh_sum[NW + 1];
  __shared__ int64_t sh_base;
  __shared__ int sh_seq;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int B = p.c.num_seqs, items = p.c.Hkv * p.chunks;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&full[i], 2);  // the copies' transaction, and the tiles' scales
      mbar_init(&empty[i], NW);
    }
    fence_barrier_init();
  }

  // ---- where this CTA's chunks begin: prefix sums of the sequences' places ----
  const int seg = (B + THREADS - 1) / THREADS;
  const int s_lo = min(B, tid * seg), s_hi = min(B, s_lo + seg);
  int64_t mine = 0;
  for (int s = s_lo; s < s_hi; ++s) mine += kv8_places<CH>(kv8_ctx(p, s));
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  if (lane == 31) sh_sum[warp] = incl;
  __syncthreads();
  int64_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w <= NW; ++w) {
    if (w < warp) before += sh_sum[w];
    total += sh_sum[w];
  }
  const int64_t U = total * items;
  // (no more shares than places, so that an item's parts lie in consecutive CTAs)
  const int64_t n_cta = min(static_cast<int64_t>(gridDim.x), max(U, int64_t{1}));
  const int64_t u0 = min(U, U * blockIdx.x / n_cta);
  u1 = min(U, U * (blockIdx.x + 1) / n_cta);
  if (tid == 0 && blockIdx.x == 0) *p.places = U;
  before += incl - mine;  // places (of one item) before this thread's sequences
  if (u0 < U && mine > 0 && before * items <= u0 && u0 < (before + mine) * items) {
    int s = s_lo;
    int64_t b = before;
    for (;; ++s) {
      const int64_t n = kv8_places<CH>(kv8_ctx(p, s));
      if (u0 < (b + n) * items) break;
      b += n;
    }
    sh_seq = s;
    sh_base = b * items;
  }
  __syncthreads();

  // sequences without a key: zeros (their rows belong to no chunk)
  for (int s = blockIdx.x; s < B; s += gridDim.x) {
    if (kv8_ctx(p, s) > 0) continue;
    for (int e = tid; e < p.Lq * p.H * p.c.D; e += THREADS) {
      const int d = e % p.c.D, h = e / p.c.D % p.H, i = e / p.c.D / p.H;
      static_cast<uint16_t*>(p.out)[s * p.so[0] + i * p.so[1] + h * p.so[2] + d * p.so[3]] = 0;
    }
    for (int e = tid; e < p.Lq * p.H; e += THREADS)
      if (p.lse) p.lse[static_cast<int64_t>(s) * p.Lq * p.H + e] = -INFINITY;
  }
  if (u0 >= u1) {
    if (tid == 0) p.bound[blockIdx.x] = make_int4(0, 0, 0, 0);
    return false;
  }
  w0.s = sh_seq;
  w0.load(p);
  w0.at = u0;
  w0.r = static_cast<int>((u0 - sh_base) / (w0.n + kItemCost));
  w0.j = static_cast<int>((u0 - sh_base) % (w0.n + kItemCost));
  if (w0.j >= w0.n) w0.next_item(p, items);  // u0 lies on an item's empty places
  const bool any = w0.live(p, u1);
  if (tid == 0) p.bound[blockIdx.x] = any ? make_int4(w0.s, w0.r, w0.j, w0.n) : make_int4(0, 0, 0, 0);
  return any;
}

// The producer warp of both kernels.
template <class C>
__device__ __forceinline__ void kv8_produce(const Kv8TcParams& p, const CUtensorMap& tmK, const CUtensorMap& tmV, uint8_t* smem,
                                            uint64_t* full, uint64_t* empty, const Kv8Walk<C::CH>& w0, int64_t u1) {
  constexpr int CH = C::CH, NT = C::NT, NS = C::NS, RT = C::RT;
  const int lane = threadIdx.x & 31, items = p.c.Hkv * p.chunks;
  float* meta = reinterpret_cast<float*>(smem + C::META_OFF);
  // lane t < NT looks after tile t of a chunk: its page and scales are loaded
  // one and two chunks ahead, so that no chunk waits on them
  tma_prefetch_desc(&tmK);
  tma_prefetch_desc(&tmV);
  const int nbox = CH / p.box_rows, tiles_per_box = p.box_rows / 16;
  struct Meta { int64_t page; int row, kvh, ctx, tok0; float ks, vs; };
  bool wide = false;  // a V scale of the item, up to this chunk, lies beyond 2^kFar
  auto fetch_page = [&](const Kv8Walk<CH>& w, bool live) {
    Meta m{};
    m.page = -1;
    m.ctx = w.ctx;
    m.tok0 = w.j * CH;
    m.kvh = w.r / p.chunks;
    const int tok = m.tok0 + lane * 16;
    if (live && lane < NT && tok < w.ctx) {
      const int lp = tok / p.c.P;
      m.row = tok - lp * p.c.P;
      m.page = p.c.block_tables[w.s * p.c.sbt[0] + lp * p.c.sbt[1]];
    }
    return m;
  };
  auto fetch_scales = [&](Meta& m) {
    m.ks = m.vs = 0.f;
    if (m.page >= 0 && m.page < p.c.num_blocks) {
      const int g = m.row / p.c.group;
      m.ks = *kv8_scale(p.c.plane[0], m.page, m.kvh, g);
      m.vs = *kv8_scale(p.c.plane[1], m.page, m.kvh, g);
    }
  };
  Kv8Walk<CH> w = w0;
  bool more = true, more2;  // chunks one and two ahead
  int issued = 0;           // chunks whose copies were started
  Meta cur = fetch_page(w, true);
  w.next(p, items);
  more = w.live(p, u1);
  Meta nxt = fetch_page(w, more);
  fetch_scales(cur);
  for (int it = 0;; ++it) {
    more2 = more;
    if (more) {
      w.next(p, items);
      more2 = w.live(p, u1);
      if (more2 && w.j == 0) {  // an item begins two chunks ahead: its query rows to L2
        const int kvh = w.r / p.chunks, row0 = (w.r - kvh * p.chunks) * RT, lines = C::PLANE / CH / 64;
        for (int e = lane; e < RT * lines; e += 32) {
          const int row = row0 + e / lines, d = e % lines * 64;
          if (row < p.rows && d < p.c.D)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(kv8_q_row(p, w.s, kvh, row) + d * p.sq[3]));
        }
      }
    }
    Meta far = fetch_page(w, more2);
    const int st = it % NS;
    if (it >= NS && !__all_sync(0xffffffffu, mbar_wait_sleep(&empty[st], ((it / NS) - 1) & 1))) break;
    const int boxes = min(nbox, (cur.ctx - cur.tok0 + p.box_rows - 1) / p.box_rows);
    if (lane == 0) mbar_arrive_expect_tx(&full[st], boxes * 2 * C::CB * p.box_rows * C::ROWB);
    __syncwarp();
    const int src = lane < nbox ? lane * tiles_per_box : 0;
    const int page = static_cast<int>(__shfl_sync(0xffffffffu, cur.page, src));
    const int row = __shfl_sync(0xffffffffu, cur.row, src);
    if (lane < boxes) {
      uint8_t* k = smem + st * C::STAGE + lane * p.box_rows * C::ROWB;
#pragma unroll
      for (int cb = 0; cb < C::CB; ++cb) {
        tma_load_4d(k + cb * CH * C::ROWB, &tmK, &full[st], cb * 128, row, cur.kvh, page);
        tma_load_4d(k + C::PLANE + cb * CH * C::ROWB, &tmV, &full[st], cb * 128, row, cur.kvh, page);
      }
    }
    fetch_scales(nxt);
    const bool bad = !(cur.vs < INFINITY);  // NaN or inf
    const bool past = cur.tok0 + lane * 16 >= cur.ctx;  // no key: a scale like any other's
    const float v = bad || past ? 1.f : fmaxf(cur.vs, kMinVs), lv = v > kMinVs ? log2f(v) + kPBias : kMinLv;
    wide = __any_sync(0xffffffffu, lane < NT && fabsf(lv - kPBias) > kFar) || (wide && cur.tok0 > 0);
    if (lane < NT) {
      float* mt = meta + st * 3 * NT;
      mt[lane] = cur.ks;
      mt[NT + lane] = bad ? __uint_as_float(0x7fffffffu) : lv;
      mt[2 * NT + lane] = wide ? 0.f : kLBiasInv / v;
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&full[st]);
    issued = it + 1;
    if (!more) break;
    cur = nxt;
    nxt = far;
    more = more2;
  }
  // the CTA's shared memory outlives the copies into it, also where a wait ran out
  for (int it = max(0, issued - NS); it < issued; ++it) mbar_wait_sleep(&full[it % NS], (it / NS) & 1);
}

// Up to eight query rows a KV head (a decode step with up to eight query heads for
// each).  Bound by memory: 64 x <= 8192 keys of 8 heads x 128 (e4m3) in 99 us with
// the join, 5.54 TB/s, 84 % of the measured copy rate; 3 x <= 131071 keys (int8, 8
// rows, capped scores) in 99, 83 %.  Head dim 64: 74 us (57 %), 256: 218 (77 %).  What
// is missing is the first data's way (4 us) and the end, where the CTAs finish within
// 10 % of each other.  Steps on the way, both cases: rows on the MMA's M side, 4 or 8
// of its 16 real, 139 and 148 us; with three CTAs an SM, Q in shared memory, 120 and
// 133; keys on the M side 99 and 100 without the join.  One request of 777 keys takes 10.2 us: two launches and the chain
// of context, page, codes, join.
template <int CODE, int DP>
__global__ void __launch_bounds__(Kv8Few<DP>::THREADS, Kv8Few<DP>::CTAS)
    kv8_attention_few_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                             const __grid_constant__ Kv8TcParams p) {
  using C = Kv8Few<DP>;
  constexpr int NW = C::NW, CH = C::CH, NT = C::NT, TP = C::TP, NS = C::NS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const float* meta = reinterpret_cast<const float*>(smem + C::META_OFF);
  float* obuf = reinterpret_cast<float*>(smem + C::OBUF_OFF);
  float* mlbuf = reinterpret_cast<float*>(smem + C::ML_OFF);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
  uint64_t* empty = full + NS;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int items = p.c.Hkv * p.chunks;
  Kv8Walk<CH> w0;
  int64_t u1;
  __shared__ int sh_fail;
  if (tid == 0) sh_fail = 0;
  if (!kv8_begin<C>(p, full, empty, w0, u1)) return;
  if (warp == NW) {
    kv8_produce<C>(p, tmK, tmV, smem, full, empty, w0, u1);
    return;
  }

  // ---------------- consumers ----------------
  const int g = lane >> 2, t4 = lane & 3, mi = lane >> 3, rr = lane & 7;
  const uint32_t sbase = smem_u32(smem);
  Kv8Walk<CH> w = w0;
  int it = 0;
  bool ok = true;
  while (ok && w.live(p, u1)) {
    // one item: chunks [w.j, j_end) of it are this CTA's
    const int j0 = w.j, j_end = static_cast<int>(min(static_cast<int64_t>(w.n), w.j + (u1 - w.at))), s = w.s, ctx = w.ctx;
    const int kvh = w.r / p.chunks, rc = w.r - kvh * p.chunks;

    // ---- query rows to fp16 B fragments, each row scaled by a power of two ----
    // The keys are the M side of both products (S^T = Kc Q^T, O^T = Vc^T P^T), so
    // eight query rows fill an MMA.  k order: thread t4 of a quad holds elements
    // 4 t4 .. 4 t4 + 3 of each 16, the order in which a 32-bit word of codes has them.
    uint32_t qb[DP / 16][2];
    auto to_float = [&](uint32_t raw) {
      return p.bf16 ? __uint_as_float(raw << 16) : __half2float(__ushort_as_half(static_cast<uint16_t>(raw)));
    };
    uint2 raw[DP / 16];  // all loads in flight at once
    const int row = rc * 8 + g;
    const bool real = row < p.rows;
    const uint16_t* src = kv8_q_row(p, s, kvh, real ? row : 0);
#pragma unroll
    for (int b = 0; b < DP / 16; ++b) {
      const int d = b * 16 + 4 * t4;
      uint2 v = make_uint2(0, 0);
      if (p.q_vec) {
        if (real && d < p.c.D) v = *reinterpret_cast<const uint2*>(src + d);
      } else {
        uint32_t e[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) e[k] = real && d + k < p.c.D ? src[(d + k) * p.sq[3]] : 0;
        v = make_uint2(e[0] | (e[1] << 16), e[2] | (e[3] << 16));
      }
      raw[b] = v;
    }
    // scores come out with this thread's rows 2 t4 and 2 t4 + 1 (of each eight)
    float fac[2];
    int lim[2];  // keys that a row sees
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int row = rc * 8 + 2 * t4 + k;
      lim[k] = row < p.rows ? ctx - p.Lq + row / p.G + 1 : ctx;  // rows that pad the tile see every key
    }
    float top = 0.f;
    bool odd = false;
#pragma unroll
    for (int b = 0; b < DP / 16; ++b) {
      const uint2 v = raw[b];
      const float f[4] = {to_float(v.x & 0xffff), to_float(v.x >> 16), to_float(v.y & 0xffff), to_float(v.y >> 16)};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        top = fmaxf(top, fabsf(f[k]));
        odd |= !(fabsf(f[k]) < INFINITY);
      }
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    odd |= __shfl_xor_sync(0xffffffffu, odd, 1);
    odd |= __shfl_xor_sync(0xffffffffu, odd, 2);
    // 2^e <= top < 2^(e+1); the row's largest comes to [2^8, 2^9)
    const int e2 = odd || top == 0.f ? 8 : max(-110, static_cast<int>(__float_as_uint(top) >> 23) - 127);
    const float up = __uint_as_float(static_cast<uint32_t>(127 + 8 - e2) << 23);
    const float f = p.scale * __uint_as_float(static_cast<uint32_t>(127 - 8 + e2) << 23);
    fac[0] = __shfl_sync(0xffffffffu, f, 8 * t4);
    fac[1] = __shfl_sync(0xffffffffu, f, 8 * t4 + 4);
#pragma unroll
    for (int b = 0; b < DP / 16; ++b) {
      const uint2 v = raw[b];
      const uint32_t q01 = Elem<__half>::pack2(to_float(v.x & 0xffff) * up, to_float(v.x >> 16) * up);
      const uint32_t q23 = Elem<__half>::pack2(to_float(v.y & 0xffff) * up, to_float(v.y >> 16) * up);
      qb[b][0] = q01;
      qb[b][1] = q23;
    }

    float o[DP / 16][4];  // (column 2 g, 2 g + 1 of each 16) x (row 2 t4, 2 t4 + 1): c0 c1 / c2 c3
    float m[2], l[2];
    int above[2];   // keys counted in fp16's normal range since the maximum last rose
    bool many = false;  // every row of the warp has kFew of them
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      m[k] = kNoMax;
      l[k] = 0.f;
      above[k] = 0;
    }
    // this thread's first row of the stored scores, [item][eight rows of each chunk of rows][score_ld]
    float* const score_row = p.scores + ((static_cast<int64_t>(s) * items + w.r) * 8 + 2 * t4) * p.score_ld;
    const int open = ctx - p.Lq + 1;  // keys below it are seen by every row

    for (int j = j0; j < j_end; ++j, ++it) {
      const int st = it % NS;
      if (!mbar_wait(&full[st], (it / NS) & 1)) {
        sh_fail = 1;  // read by all warps after the next barrier: they leave together
        break;
      }
      const uint32_t kbase = sbase + st * C::STAGE, vbase = kbase + C::PLANE;
      const float* mt = meta + st * 3 * NT;
      const int t = warp * TP, tok = j * CH + t * 16, r0 = t * 16;
      if (tok < ctx) {
        if (CODE == kE4M3 && tok + 16 * TP > ctx) {
          // rows past the end may hold NaN codes: zero their V rows (several
          // warps may write the same zeros)
          uint8_t* vt = smem + st * C::STAGE + C::PLANE;
          for (int i = lane; i < 16 * TP * C::CB * (C::ROWB / 16); i += 32) {
            const int r = i / (C::CB * (C::ROWB / 16)), cc = i % (C::CB * (C::ROWB / 16));
            if (tok + r >= ctx)
              *reinterpret_cast<uint4*>(vt + (cc / 8) * CH * C::ROWB + kv8_sw<DP>(r0 + r, cc % 8)) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        // ---- S^T = Kc Q^T for TP tiles of 16 keys ----
        float x[TP][4];  // c0 c1: key g, rows 2 t4, 2 t4 + 1; c2 c3: key g + 8
#pragma unroll
        for (int u = 0; u < TP; ++u) x[u][0] = x[u][1] = x[u][2] = x[u][3] = 0.f;
#pragma unroll
        for (int kb = 0; kb < DP / 32; ++kb) {
          const int piece = 2 * kb + (mi >> 1);
          uint32_t r[TP][4];
#pragma unroll
          for (int u = 0; u < TP; ++u)
            ldsm_x4(kbase + (piece >> 3) * CH * C::ROWB + kv8_sw<DP>(r0 + u * 16 + (mi & 1) * 8 + rr, piece & 7), r[u][0],
                    r[u][1], r[u][2], r[u][3]);
#pragma unroll
          for (int k = 0; k < 2; ++k) {  // k16 step; r[.][2 k]: the first eight keys, r[.][2 k + 1]: the others
#pragma unroll
            for (int u = 0; u < TP; ++u) {
              uint32_t af[4];
              codes_to_half<CODE, 0>(r[u][2 * k], af[0], af[2]);
              codes_to_half<CODE, 0>(r[u][2 * k + 1], af[1], af[3]);
              Mma<__half>::run(x[u], af, qb[2 * kb + k][0], qb[2 * kb + k][1]);
            }
          }
        }
        // ---- scores, base 2 ----
        const bool masked = tok + 16 * TP > open;
        float lv[TP], ivs[TP], y[2] = {-INFINITY, -INFINITY};  // y: largest score + log2 vs + kPBias
#pragma unroll
        for (int u = 0; u < TP; ++u) {
          const float ks = mt[t + u];
          lv[u] = mt[NT + t + u];
          ivs[u] = mt[2 * NT + t + u];
          const float f0 = fac[0] * ks, f1 = fac[1] * ks;
          x[u][0] *= f0;
          x[u][1] *= f1;
          x[u][2] *= f0;
          x[u][3] *= f1;
        }
        bool v_bad = lv[0] != lv[0];  // (the tiles of a NaN or infinite V scale are marked by a NaN)
        if (TP > 1) v_bad |= lv[TP - 1] != lv[TP - 1];
        if (v_bad) {
#pragma unroll
          for (int u = 0; u < TP; ++u) lv[u] = lv[u] == lv[u] ? lv[u] : kPBias;
        }
        if (p.inv_cap > 0.f) {
#pragma unroll
          for (int u = 0; u < TP; ++u) kv8_cap(x[u], p.inv_cap, p.cap2);
        }
        if (masked) {
#pragma unroll
          for (int u = 0; u < TP; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (tok + u * 16 + g + (e & 2) * 4 >= lim[e & 1]) x[u][e] = -INFINITY;
        }
#pragma unroll
        for (int u = 0; u < TP; ++u)
#pragma unroll
          for (int k = 0; k < 2; ++k) y[k] = fmaxf(y[k], lv[u] + fmaxf(x[u][k], x[u][k + 2]));
        if (p.scores) {
#pragma unroll
          for (int u = 0; u < TP; ++u) {
            if (tok + u * 16 >= p.score_ld) continue;
            float* sp = score_row + tok + u * 16 + g;  // (rows that pad the tile have rows of their own there)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              sp[k * p.score_ld] = x[u][k];
              sp[k * p.score_ld + 8] = x[u][k + 2];
            }
          }
        }
        // ---- running maximum: raised only when a score passes it by 2^kLag ----
        bool up = false;
#pragma unroll
        for (int k = 0; k < 2; ++k) up |= y[k] > m[k] + (kLag + kPBias);
        if (__any_sync(0xffffffffu, up)) {
          float al[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float mx = y[k] - kPBias;
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float mn = fmaxf(m[k], mx);
            const float h = fast_exp2(0.5f * (m[k] - mn));
            al[k] = h * h;
            m[k] = mn;
            l[k] = kv8_add_down(0.f, l[k], h);
            above[k] = 0;
          }
#pragma unroll
          for (int i = 0; i < DP / 16; ++i) {
            o[i][0] *= al[0];
            o[i][1] *= al[1];
            o[i][2] *= al[0];
            o[i][3] *= al[1];
          }
          many = false;
        }
        if (ivs[0] == 0.f) {  // a scale beyond 2^kFar in this chunk or before it
#pragma unroll
          for (int u = 0; u < TP; ++u) {
#pragma unroll
            for (int e = 0; e < 4; ++e) l[e & 1] = kv8_add_term(l[e & 1], x[u][e] - m[e & 1]);
            if (lv[u] == kMinLv) lv[u] = -INFINITY;
          }
        }
        uint32_t pb[TP][2];  // P^T fragments
#pragma unroll
        for (int u = 0; u < TP; ++u)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float c0 = lv[u] - m[k];
            x[u][k] = fast_exp2(x[u][k] + c0);
            x[u][k + 2] = fast_exp2(x[u][k + 2] + c0);
            l[k] = fmaf(x[u][k] + x[u][k + 2], ivs[u], l[k]);
          }
        // ---- weights below fp16's normal range (2^-27 of the largest): while a row
        // of the warp has fewer than kFew keys above it, they go through the
        // product apart, times 2^24, so that a column in which those few keys have
        // zeros keeps its precision.  Ordinary rows pass kFew in their first step ----
        bool apart = false;
        if (!many) {
          float least = 1.f;
          int fewest = kFew;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            int n = 0;
#pragma unroll
            for (int u = 0; u < TP; ++u)
#pragma unroll
              for (int e = k; e < 4; e += 2) {
                least = fminf(least, x[u][e]);
                n += x[u][e] >= kHalfMin;
              }
            n += __shfl_xor_sync(0xffffffffu, n, 4);
            n += __shfl_xor_sync(0xffffffffu, n, 8);
            n += __shfl_xor_sync(0xffffffffu, n, 16);
            above[k] += n;
            fewest = min(fewest, above[k]);
          }
          many = __all_sync(0xffffffffu, fewest >= kFew);
          apart = !many && __any_sync(0xffffffffu, least < kHalfMin);
        }
        if (apart) {
          uint32_t pc[TP][2];
          bool some = false;
#pragma unroll
          for (int u = 0; u < TP; ++u) {
            float f[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float v = x[u][e];
              const bool small = v < kHalfMin;
              f[e] = small ? v * 16777216.f : 0.f;
              x[u][e] = small ? 0.f : v;
              some |= f[e] > 0.f;
            }
            pc[u][0] = transpose8x8(Elem<__half>::pack2(f[0], f[1]));
            pc[u][1] = transpose8x8(Elem<__half>::pack2(f[2], f[3]));
          }
          if (__any_sync(0xffffffffu, some)) {
#pragma unroll
            for (int db = 0; db < DP / 16; ++db) {
              float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int u = 0; u < TP; ++u) {
                uint32_t r[2], af[4];
                ldsm_x2_t(vbase + (db >> 3) * CH * C::ROWB + kv8_sw<DP>(r0 + u * 16 + (mi & 1) * 8 + rr, db & 7), r[0], r[1]);
                codes_to_half<CODE, 1>(r[0], af[0], af[1]);
                codes_to_half<CODE, 1>(r[1], af[2], af[3]);
                Mma<__half>::run(a, af, pc[u][0], pc[u][1]);
              }
#pragma unroll
              for (int e = 0; e < 4; ++e) o[db][e] = fmaf(a[e], 5.9604644775390625e-8f, o[db][e]);
            }
          }
        }
        if (v_bad) {  // a NaN or infinite V scale: NaN for the rows that see a key of the tile
#pragma unroll
        for (int u = 0; u < TP; ++u)
          if (mt[NT + t + u] != mt[NT + t + u]) {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[u][e] = tok + u * 16 < lim[e & 1] ? __uint_as_float(0x7fffffffu) : 0.f;
            }
        }
#pragma unroll
        for (int u = 0; u < TP; ++u) {
          pb[u][0] = transpose8x8(Elem<__half>::pack2(x[u][0], x[u][1]));
          pb[u][1] = transpose8x8(Elem<__half>::pack2(x[u][2], x[u][3]));
        }
        // ---- O^T += Vc^T P^T: words transposed by the load pair two keys of columns
        // 2 g and 2 g + 1, which become rows g and g + 8 of the MMA ----
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) {
          const int piece = 2 * db + (mi >> 1);
#pragma unroll
          for (int u = 0; u < TP; ++u) {
            uint32_t r[4];
            ldsm_x4_t(vbase + (piece >> 3) * CH * C::ROWB + kv8_sw<DP>(r0 + u * 16 + (mi & 1) * 8 + rr, piece & 7), r[0], r[1],
                      r[2], r[3]);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              uint32_t af[4];
              codes_to_half<CODE, 1>(r[2 * k], af[0], af[1]);
              codes_to_half<CODE, 1>(r[2 * k + 1], af[2], af[3]);
              Mma<__half>::run(o[2 * db + k], af, pb[u][0], pb[u][1]);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
    }

    // ---- join the warps that shared the rows, then finish or store a part ----
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      l[k] += __shfl_xor_sync(0xffffffffu, l[k], 4);
      l[k] += __shfl_xor_sync(0xffffffffu, l[k], 8);
      l[k] += __shfl_xor_sync(0xffffffffu, l[k], 16);
    }
    const bool whole = j0 == 0 && j_end == w.n;
    const int64_t slot = (static_cast<int64_t>(blockIdx.x) * 2 + (j0 == 0 ? 1 : 0)) * 8;
#pragma unroll
    for (int dh = 0; dh < DP / C::DH; ++dh) {
      asm volatile("bar.sync 1, %0;" ::"n"(NW * 32) : "memory");  // the buffer is free again
#pragma unroll
      for (int i = 0; i < C::DH / 16; ++i) {
        const float* ot = o[dh * (C::DH / 16) + i];
        float* dst = obuf + (warp * 8 + 2 * t4) * C::OLD + i * 16 + 2 * g;
        *reinterpret_cast<float2*>(dst) = make_float2(ot[0], ot[2]);
        *reinterpret_cast<float2*>(dst + C::OLD) = make_float2(ot[1], ot[3]);
      }
      if (dh == 0 && g == 0) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
          *reinterpret_cast<float2*>(mlbuf + (warp * 8 + 2 * t4 + k) * 2) = make_float2(m[k], l[k]);
      }
      asm volatile("bar.sync 1, %0;" ::"n"(NW * 32) : "memory");
      for (int e = tid; e < 8 * (C::DH / 4); e += NW * 32) {
        const int row = e / (C::DH / 4), d = (e - row * (C::DH / 4)) * 4;
        const int grow = rc * 8 + row;
        if (grow >= p.rows) continue;
        float M = -INFINITY;
#pragma unroll
        for (int k = 0; k < NW; ++k) M = fmaxf(M, mlbuf[(k * 8 + row) * 2]);
        const float Mu = M == -INFINITY ? 0.f : M;
        float L = 0.f;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < NW; ++k) {
          const int at = k * 8 + row;
          const float hf = fast_exp2(0.5f * (mlbuf[at * 2] - Mu)), f = hf * hf;
          L = kv8_add_down(L, mlbuf[at * 2 + 1], hf);
          const float4 v = *reinterpret_cast<const float4*>(obuf + at * C::OLD + d);
          a.x = fmaf(v.x, f, a.x);
          a.y = fmaf(v.y, f, a.y);
          a.z = fmaf(v.z, f, a.z);
          a.w = fmaf(v.w, f, a.w);
        }
        const int dd = dh * C::DH + d;
        if (whole) {
          const int i = grow / p.G, h = kvh * p.G + grow - i * p.G;
          const float2 over = kv8_over(L);
          uint16_t* out = static_cast<uint16_t*>(p.out) + s * p.so[0] + i * p.so[1] + h * p.so[2];
          const float f[4] = {a.x * over.x * over.y, a.y * over.x * over.y, a.z * over.x * over.y, a.w * over.x * over.y};
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (dd + k < p.c.D)
              out[(dd + k) * p.so[3]] = p.bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(f[k])) : __half_as_ushort(__float2half_rn(f[k]));
          if (dd == 0) {
            const float v = L != 0.f ? M + kLBias + log2f(L) : -INFINITY;
            if (p.lse) p.lse[(static_cast<int64_t>(s) * p.Lq + i) * p.H + h] = v * kLn2;
            if (p.lse2) p.lse2[(static_cast<int64_t>(s) * p.c.Hkv + kvh) * p.rows + grow] = v;
          }
        } else {
          *reinterpret_cast<float4*>(p.part_o + (slot + row) * DP + dd) = a;
          if (dd == 0) *reinterpret_cast<float2*>(p.part_ml + (slot + row) * 2) = make_float2(M, L);
        }
      }
    }
    ok = *static_cast<volatile int*>(&sh_fail) == 0;
    // the next item
    w.next_item(p, items);
  }
}

// 16 and 32 query rows.  Bound by the issue slots and latencies of the conversions and
// MMAs (two consumer warps a scheduler): 64 x <= 8192 keys of 8 heads, 32 rows, in 203
// us, 16 rows in 125 (head dim 64: 154 and 103; 256: 381 and 249); 24 x <= 6000 keys of
// 4 heads, 32 rows (int8), in 49, 65 with the weights.  The branch for V scales far
// apart costs 32 rows up to 9 us of that: as a loop of its own it spilled (252 us for
// the first), with its sums in shared memory it took 207.  Where each warp held eight rows and walked all keys, every code was
// converted once for each warp (57 and 69 us, then against 47 and 61).  Chunks of 64 keys with three CTAs an SM
// took 251 us for the first, 61 without weights for the last.
template <int CODE, int DP, int NR>
__global__ void __launch_bounds__(Kv8Many<DP, NR>::THREADS, Kv8Many<DP, NR>::CTAS)
    kv8_attention_many_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                              const __grid_constant__ Kv8TcParams p) {
  using C = Kv8Many<DP, NR>;
  constexpr int NW = C::NW, CH = C::CH, NT = C::NT, TP = C::TP, NS = C::NS, RT = C::RT, MB = C::MB;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const float* meta = reinterpret_cast<const float*>(smem + C::META_OFF);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
  uint64_t* empty = full + NS;
  uint2* const qf = reinterpret_cast<uint2*>(smem + C::Q_OFF);
  uint2* const pf = reinterpret_cast<uint2*>(smem + C::P_OFF);
  uint2* const pf2 = pf + NT * NR * 32;
  float* const sfac = reinterpret_cast<float*>(smem + C::FAC_OFF);
  float* const smax = reinterpret_cast<float*>(smem + C::MAX_OFF);
  volatile int* const flag_up = reinterpret_cast<volatile int*>(smem + C::FLAG_OFF);
  volatile int* const flag_apart = flag_up + NW;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int items = p.c.Hkv * p.chunks;
  Kv8Walk<CH> w0;
  int64_t u1;
  if (!kv8_begin<C>(p, full, empty, w0, u1)) return;
  if (warp == NW) {
    kv8_produce<C>(p, tmK, tmV, smem, full, empty, w0, u1);
    return;
  }

  // ---------------- consumers ----------------
  auto bar = [] { asm volatile("bar.sync 1, %0;" ::"n"(NW * 32) : "memory"); };
  const int g = lane >> 2, t4 = lane & 3, mi = lane >> 3, rr = lane & 7;
  const uint32_t sbase = smem_u32(smem);
  Kv8Walk<CH> w = w0;
  int it = 0;
  bool ok = true;
  while (ok && w.live(p, u1)) {
    const int j0 = w.j, j_end = static_cast<int>(min(static_cast<int64_t>(w.n), w.j + (u1 - w.at))), s = w.s, ctx = w.ctx;
    const int kvh = w.r / p.chunks, rc = w.r - kvh * p.chunks;

    // ---- query rows to fp16 B fragments in shared memory, as in the other kernel:
    // warp w makes those of rows 8 w .. 8 w + 7 ----
    if (warp < NR) {
      auto to_float = [&](uint32_t raw) {
        return p.bf16 ? __uint_as_float(raw << 16) : __half2float(__ushort_as_half(static_cast<uint16_t>(raw)));
      };
      uint2 raw[DP / 16];
      const int row = rc * RT + warp * 8 + g;
      const bool real = row < p.rows;
      const uint16_t* src = kv8_q_row(p, s, kvh, real ? row : 0);
      float top = 0.f;
      bool odd = false;
#pragma unroll
      for (int b = 0; b < DP / 16; ++b) {
        const int d = b * 16 + 4 * t4;
        uint2 v = make_uint2(0, 0);
        if (p.q_vec) {
          if (real && d < p.c.D) v = *reinterpret_cast<const uint2*>(src + d);
        } else {
          uint32_t e[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) e[k] = real && d + k < p.c.D ? src[(d + k) * p.sq[3]] : 0;
          v = make_uint2(e[0] | (e[1] << 16), e[2] | (e[3] << 16));
        }
        raw[b] = v;
      }
#pragma unroll
      for (int b = 0; b < DP / 16; ++b) {
        const uint2 v = raw[b];
        const float f[4] = {to_float(v.x & 0xffff), to_float(v.x >> 16), to_float(v.y & 0xffff), to_float(v.y >> 16)};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          top = fmaxf(top, fabsf(f[k]));
          odd |= !(fabsf(f[k]) < INFINITY);
        }
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      odd |= __shfl_xor_sync(0xffffffffu, odd, 1);
      odd |= __shfl_xor_sync(0xffffffffu, odd, 2);
      const int e2 = odd || top == 0.f ? 8 : max(-110, static_cast<int>(__float_as_uint(top) >> 23) - 127);
      const float up = __uint_as_float(static_cast<uint32_t>(127 + 8 - e2) << 23);
      if (t4 == 0) sfac[warp * 8 + g] = p.scale * __uint_as_float(static_cast<uint32_t>(127 - 8 + e2) << 23);
#pragma unroll
      for (int b = 0; b < DP / 16; ++b) {
        const uint2 v = raw[b];
        qf[(b * NR + warp) * 32 + lane] = make_uint2(Elem<__half>::pack2(to_float(v.x & 0xffff) * up, to_float(v.x >> 16) * up),
                                                     Elem<__half>::pack2(to_float(v.y & 0xffff) * up, to_float(v.y >> 16) * up));
      }
    }
    bar();
    // this thread's rows are 2 t4 and 2 t4 + 1 of each eight.  (What is needed once a
    // chunk or less is looked up or worked out again: held, it would spill.)
    auto limit = [&](int n, int k) {  // keys that a row sees; rows that pad the tile see every key
      const int row = rc * RT + n * 8 + 2 * t4 + k;
      return row < p.rows ? ctx - p.Lq + row / p.G + 1 : ctx;
    };
    float o[MB][NR][4];  // (column 2 g, 2 g + 1 of each 16 of the warp's) x (row 2 t4, 2 t4 + 1)
    float m[NR][2], l[NR][2];  // the maximum is the CTA's, the sum this thread's keys'
    uint32_t above[NR] = {};  // two counts of keys in fp16's normal range since the maximum last rose, 16 bits each
    bool many = false;
#pragma unroll
    for (int n = 0; n < NR; ++n) {
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) o[mb][n][0] = o[mb][n][1] = o[mb][n][2] = o[mb][n][3] = 0.f;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        m[n][k] = kNoMax;
        l[n][k] = 0.f;
      }
    }
    float* const score_row = p.scores + ((static_cast<int64_t>(s) * items + w.r) * RT + 2 * t4) * p.score_ld;
    const int open = ctx - p.Lq + 1;  // keys below it are seen by every row

    for (int j = j0; j < j_end; ++j, ++it) {
      const int st = it % NS;
      const bool arrived = mbar_wait(&full[st], (it / NS) & 1);
      const uint32_t kbase = sbase + st * C::STAGE, vbase = kbase + C::PLANE;
      const float* mt = meta + st * 3 * NT;
      const int t = warp * TP, tok = j * CH + t * 16, r0 = t * 16;
      float x[TP][NR][4], lv[TP], ivs[TP], y[NR][2];
      bool v_bad = false;
#pragma unroll
      for (int n = 0; n < NR; ++n) y[n][0] = y[n][1] = -INFINITY;
      if (arrived && tok < ctx) {
        if (CODE == kE4M3 && tok + 16 * TP > ctx) {
          // rows past the end may hold NaN codes: zero their V rows
          uint8_t* vt = smem + st * C::STAGE + C::PLANE;
          for (int i = lane; i < 16 * TP * C::CB * (C::ROWB / 16); i += 32) {
            const int r = i / (C::CB * (C::ROWB / 16)), cc = i % (C::CB * (C::ROWB / 16));
            if (tok + r >= ctx)
              *reinterpret_cast<uint4*>(vt + (cc / 8) * CH * C::ROWB + kv8_sw<DP>(r0 + r, cc % 8)) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
#pragma unroll
        for (int u = 0; u < TP; ++u)
#pragma unroll
          for (int n = 0; n < NR; ++n) x[u][n][0] = x[u][n][1] = x[u][n][2] = x[u][n][3] = 0.f;
#pragma unroll
        for (int kb = 0; kb < DP / 32; ++kb) {
          const int piece = 2 * kb + (mi >> 1);
          uint32_t r[TP][4];
#pragma unroll
          for (int u = 0; u < TP; ++u)
            ldsm_x4(kbase + (piece >> 3) * CH * C::ROWB + kv8_sw<DP>(r0 + u * 16 + (mi & 1) * 8 + rr, piece & 7), r[u][0],
                    r[u][1], r[u][2], r[u][3]);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            uint2 q[NR];
#pragma unroll
            for (int n = 0; n < NR; ++n) q[n] = qf[((2 * kb + k) * NR + n) * 32 + lane];
#pragma unroll
            for (int u = 0; u < TP; ++u) {
              uint32_t af[4];
              codes_to_half<CODE, 0>(r[u][2 * k], af[0], af[2]);
              codes_to_half<CODE, 0>(r[u][2 * k + 1], af[1], af[3]);
#pragma unroll
              for (int n = 0; n < NR; ++n) Mma<__half>::run(x[u][n], af, q[n].x, q[n].y);
            }
          }
        }
        // ---- scores, base 2 ----
        const bool masked = tok + 16 * TP > open;
#pragma unroll
        for (int u = 0; u < TP; ++u) {
          const float ks = mt[t + u];
          lv[u] = mt[NT + t + u];
          ivs[u] = mt[2 * NT + t + u];
          v_bad |= lv[u] != lv[u];
#pragma unroll
          for (int n = 0; n < NR; ++n) {
            const float2 f = *reinterpret_cast<const float2*>(sfac + n * 8 + 2 * t4);
            const float f0 = f.x * ks, f1 = f.y * ks;
            x[u][n][0] *= f0;
            x[u][n][1] *= f1;
            x[u][n][2] *= f0;
            x[u][n][3] *= f1;
          }
        }
        if (v_bad) {
#pragma unroll
          for (int u = 0; u < TP; ++u) lv[u] = lv[u] == lv[u] ? lv[u] : kPBias;
        }
        if (p.inv_cap > 0.f) {
#pragma unroll
          for (int u = 0; u < TP; ++u)
#pragma unroll
            for (int n = 0; n < NR; ++n) kv8_cap(x[u][n], p.inv_cap, p.cap2);
        }
        if (masked) {
#pragma unroll
          for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int lim = limit(n, k);
#pragma unroll
              for (int u = 0; u < TP; ++u) {
                if (tok + u * 16 + g >= lim) x[u][n][k] = -INFINITY;
                if (tok + u * 16 + g + 8 >= lim) x[u][n][k + 2] = -INFINITY;
              }
            }
        }
#pragma unroll
        for (int u = 0; u < TP; ++u)
#pragma unroll
          for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int k = 0; k < 2; ++k) y[n][k] = fmaxf(y[n][k], lv[u] + fmaxf(x[u][n][k], x[u][n][k + 2]));
        if (p.scores) {
#pragma unroll
          for (int u = 0; u < TP; ++u) {
            if (tok + u * 16 >= p.score_ld) continue;
            float* sp = score_row + tok + u * 16 + g;
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                sp[(n * 8 + k) * p.score_ld] = x[u][n][k];
                sp[(n * 8 + k) * p.score_ld + 8] = x[u][n][k + 2];
              }
          }
        }
      }
      // ---- running maximum, common to the warps: raised when a score of any of
      // them passes it by 2^kLag ----
      bool up = false;
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int k = 0; k < 2; ++k) up |= y[n][k] > m[n][k] + (kLag + kPBias);
      up = __any_sync(0xffffffffu, up);
      if (lane == 0) flag_up[warp] = (up ? 1 : 0) | (arrived ? 0 : 2);
      bar();  // also: every warp has read the last chunk's P
      int any_up = 0;
#pragma unroll
      for (int i = 0; i < NW; ++i) any_up |= flag_up[i];
      if (any_up & 2) {  // a wait ran out: all leave together, no warp waits for one that left
        ok = false;
        break;
      }
      if (any_up) {
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float mx = y[n][k] - kPBias;
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            if (g == 0) smax[warp * RT + n * 8 + 2 * t4 + k] = mx;
          }
        bar();
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          float al[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float mn = m[n][k];
#pragma unroll
            for (int i = 0; i < NW; ++i) mn = fmaxf(mn, smax[i * RT + n * 8 + 2 * t4 + k]);
            const float h = fast_exp2(0.5f * (m[n][k] - mn));
            al[k] = h * h;
            m[n][k] = mn;
            l[n][k] = kv8_add_down(0.f, l[n][k], h);
          }
          above[n] = 0;
#pragma unroll
          for (int mb = 0; mb < MB; ++mb) {
            o[mb][n][0] *= al[0];
            o[mb][n][1] *= al[1];
            o[mb][n][2] *= al[0];
            o[mb][n][3] *= al[1];
          }
        }
        many = false;
      }
      // ---- this warp's weights, as P^T fragments for everyone ----
      bool apart = false;
      if (tok < ctx) {
        if (ivs[0] == 0.f) {  // a scale beyond 2^kFar in this chunk or before it
#pragma unroll
          for (int u = 0; u < TP; ++u) {
            const float lz = lv[u] == kMinLv ? -INFINITY : lv[u];
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                l[n][e & 1] = kv8_add_term(l[n][e & 1], x[u][n][e] - m[n][e & 1]);
                x[u][n][e] = fast_exp2(x[u][n][e] + (lz - m[n][e & 1]));
              }
          }
        } else {
#pragma unroll
          for (int u = 0; u < TP; ++u)
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const float c0 = lv[u] - m[n][k];
                x[u][n][k] = fast_exp2(x[u][n][k] + c0);
                x[u][n][k + 2] = fast_exp2(x[u][n][k + 2] + c0);
                l[n][k] = fmaf(x[u][n][k] + x[u][n][k + 2], ivs[u], l[n][k]);
              }
        }
        if (!many) {  // weights below fp16's normal range go apart, as in the other kernel
          float least = 1.f;
          int fewest = kFew;
#pragma unroll
          for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              int c = 0;
#pragma unroll
              for (int u = 0; u < TP; ++u)
#pragma unroll
                for (int e = k; e < 4; e += 2) {
                  least = fminf(least, x[u][n][e]);
                  c += x[u][n][e] >= kHalfMin;
                }
              c += __shfl_xor_sync(0xffffffffu, c, 4);
              c += __shfl_xor_sync(0xffffffffu, c, 8);
              c += __shfl_xor_sync(0xffffffffu, c, 16);
              if ((above[n] >> (16 * k) & 0xffffu) < kFew) above[n] += static_cast<uint32_t>(c) << (16 * k);
              fewest = min(fewest, static_cast<int>(above[n] >> (16 * k) & 0xffffu));
            }
          many = __all_sync(0xffffffffu, fewest >= kFew);
          apart = !many && __any_sync(0xffffffffu, least < kHalfMin);
          if (apart) {
#pragma unroll
            for (int u = 0; u < TP; ++u)
#pragma unroll
              for (int n = 0; n < NR; ++n) {
                float f[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float v = x[u][n][e];
                  const bool small = v < kHalfMin;
                  f[e] = small ? v * 16777216.f : 0.f;
                  x[u][n][e] = small ? 0.f : v;
                }
                const uint32_t a = transpose8x8(Elem<__half>::pack2(f[0], f[1])), b = transpose8x8(Elem<__half>::pack2(f[2], f[3]));
                pf2[((t + u) * NR + n) * 32 + lane] = make_uint2(a, b);
              }
          }
        }
        if (v_bad) {  // a NaN or infinite V scale: NaN for the rows that see a key of the tile
#pragma unroll
          for (int u = 0; u < TP; ++u)
            if (mt[NT + t + u] != mt[NT + t + u]) {
#pragma unroll
              for (int n = 0; n < NR; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[u][n][e] = tok + u * 16 < limit(n, e & 1) ? __uint_as_float(0x7fffffffu) : 0.f;
            }
        }
#pragma unroll
        for (int u = 0; u < TP; ++u)
#pragma unroll
          for (int n = 0; n < NR; ++n) {
            const uint32_t a = transpose8x8(Elem<__half>::pack2(x[u][n][0], x[u][n][1]));
            const uint32_t b = transpose8x8(Elem<__half>::pack2(x[u][n][2], x[u][n][3]));
            pf[((t + u) * NR + n) * 32 + lane] = make_uint2(a, b);
          }
      }
      if (lane == 0) flag_apart[warp] = apart;
      bar();
      // ---- O^T += Vc^T P^T over all the chunk's tiles, this warp's columns ----
      const int tiles = min(NT, (ctx - j * CH + 16 * TP - 1) / (16 * TP) * TP);  // tiles whose P was written
      const int col0 = warp * (C::CW / 16);  // first 16-byte piece
      auto product = [&](int tile, const uint2* frag, float (&acc)[MB][NR][4]) {
        uint2 pr[NR];
#pragma unroll
        for (int n = 0; n < NR; ++n) pr[n] = frag[(tile * NR + n) * 32 + lane];
        uint32_t r[2 * MB];
        if (MB == 2) {
          const int piece = col0 + (mi >> 1);
          ldsm_x4_t(vbase + (piece >> 3) * CH * C::ROWB + kv8_sw<DP>(tile * 16 + (mi & 1) * 8 + rr, piece & 7), r[0], r[1],
                    r[2 * MB - 2], r[2 * MB - 1]);
        } else {
          ldsm_x2_t(vbase + (col0 >> 3) * CH * C::ROWB + kv8_sw<DP>(tile * 16 + (mi & 1) * 8 + rr, col0 & 7), r[0], r[1]);
        }
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          uint32_t af[4];
          codes_to_half<CODE, 1>(r[2 * mb], af[0], af[1]);
          codes_to_half<CODE, 1>(r[2 * mb + 1], af[2], af[3]);
#pragma unroll
          for (int n = 0; n < NR; ++n) Mma<__half>::run(acc[mb][n], af, pr[n].x, pr[n].y);
        }
      };
      int any_apart = 0;
#pragma unroll
      for (int i = 0; i < NW; ++i) any_apart |= flag_apart[i] << i;
      if (any_apart) {
        float a[MB][NR][4];
#pragma unroll
        for (int i = 0; i < MB * NR * 4; ++i) a[i / (NR * 4)][i / 4 % NR][i % 4] = 0.f;
#pragma unroll 1
        for (int tile = 0; tile < tiles; ++tile)
          if ((any_apart >> (tile / TP)) & 1) product(tile, pf2, a);
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
          for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[mb][n][e] = fmaf(a[mb][n][e], 5.9604644775390625e-8f, o[mb][n][e]);
      }
      if (tiles == NT) {
#pragma unroll
        for (int tile = 0; tile < NT; ++tile) product(tile, pf, o);
      } else {
#pragma unroll 1
        for (int tile = 0; tile < tiles; ++tile) product(tile, pf, o);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
    }

    // ---- the warps' sums, then each warp finishes or stores its columns ----
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float v = l[n][k];
        v += __shfl_xor_sync(0xffffffffu, v, 4);
        v += __shfl_xor_sync(0xffffffffu, v, 8);
        v += __shfl_xor_sync(0xffffffffu, v, 16);
        l[n][k] = v;
      }
    bar();  // the last maxima have been read
    if (g == 0) {
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int k = 0; k < 2; ++k) smax[warp * RT + n * 8 + 2 * t4 + k] = l[n][k];
    }
    bar();
    const bool whole = j0 == 0 && j_end == w.n;
    const int64_t slot = (static_cast<int64_t>(blockIdx.x) * 2 + (j0 == 0 ? 1 : 0)) * RT;
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int row = n * 8 + 2 * t4 + k, grow = rc * RT + row;
        if (grow >= p.rows) continue;
        float L = 0.f;
#pragma unroll
        for (int i = 0; i < NW; ++i) L += smax[i * RT + row];
        const int d0 = warp * C::CW + 2 * g;
        if (whole) {
          const int i = grow / p.G, h = kvh * p.G + grow - i * p.G;
          const float2 over = kv8_over(L);
          uint16_t* out = static_cast<uint16_t*>(p.out) + s * p.so[0] + i * p.so[1] + h * p.so[2];
#pragma unroll
          for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int d = d0 + mb * 16 + c;
              const float f = o[mb][n][2 * c + k] * over.x * over.y;
              if (d < p.c.D) out[d * p.so[3]] = p.bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(f)) : __half_as_ushort(__float2half_rn(f));
            }
          if (warp == 0 && g == 0) {
            const float v = L != 0.f ? m[n][k] + kLBias + log2f(L) : -INFINITY;
            if (p.lse) p.lse[(static_cast<int64_t>(s) * p.Lq + i) * p.H + h] = v * kLn2;
            if (p.lse2) p.lse2[(static_cast<int64_t>(s) * p.c.Hkv + kvh) * p.rows + grow] = v;
          }
        } else {
#pragma unroll
          for (int mb = 0; mb < MB; ++mb)
            *reinterpret_cast<float2*>(p.part_o + (slot + row) * DP + d0 + mb * 16) = make_float2(o[mb][n][k], o[mb][n][2 + k]);
          if (warp == 0 && g == 0) *reinterpret_cast<float2*>(p.part_ml + (slot + row) * 2) = make_float2(m[n][k], L);
        }
      }
    // the next item
    w.next_item(p, items);
  }
}

// Joins the parts of the items that the split cut.  CTA (c, y) looks at the
// boundary before the main grid's CTA c: if it is the first one inside its item, it
// merges the item's parts for four query rows, in order.  The parts are those of
// CTA c - 1 (slot 1: the item begins in it) and of the CTAs from c to the one that
// holds the item's last chunk (slot 0).  A thread merges four columns of a row and
// finds the row's maximum and sum for itself, so there are two round trips to
// memory: the boundaries, then everything else.
template <int DP>
__global__ void __launch_bounds__(DP) kv8_attention_join_kernel(const __grid_constant__ Kv8TcParams p, int RT, int N) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int c = blockIdx.x + 1;
  const int4 a = p.bound[c - 1], b = p.bound[c];
  const int64_t U = *p.places;
  if (b.w == 0 || b.z == 0) return;                        // no chunk, or an item begins here
  if (a.x == b.x && a.y == b.y && a.z > 0) return;         // not the item's first cut
  const int64_t n_cta = min(static_cast<int64_t>(N), U);
  const int64_t last = U * c / n_cta + (b.w - b.z) - 1;    // place of the item's last chunk
  const int n = static_cast<int>(((last + 1) * n_cta - 1) / U) - c + 2;  // parts
  const int s = b.x, kvh = b.y / p.chunks, rc = b.y - kvh * p.chunks;
  const int r = blockIdx.y * 4 + threadIdx.x / (DP / 4), d = threadIdx.x % (DP / 4) * 4;
  const int grow = rc * RT + r;
  if (grow >= p.rows) return;
  auto slot = [&](int k) { return (static_cast<int64_t>(c - 1 + k) * 2 + (k == 0 ? 1 : 0)) * RT + r; };
  float M = kNoMax, L = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k0 = 0; k0 < n; k0 += 8) {
    float2 ml[8];
    float4 v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      ml[u] = make_float2(kNoMax, 0.f);
      v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (k0 + u < n) {
        ml[u] = *reinterpret_cast<const float2*>(p.part_ml + slot(k0 + u) * 2);
        v[u] = *reinterpret_cast<const float4*>(p.part_o + slot(k0 + u) * DP + d);
      }
    }
    float Mn = M;
#pragma unroll
    for (int u = 0; u < 8; ++u) Mn = fmaxf(Mn, ml[u].x);
    const float h0 = fast_exp2(0.5f * (M - Mn)), f0 = h0 * h0;
    L = kv8_add_down(0.f, L, h0);
    M = Mn;
    o.x *= f0;
    o.y *= f0;
    o.z *= f0;
    o.w *= f0;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float h = fast_exp2(0.5f * (ml[u].x - M)), f = h * h;
      L = kv8_add_down(L, ml[u].y, h);
      o.x = fmaf(v[u].x, f, o.x);
      o.y = fmaf(v[u].y, f, o.y);
      o.z = fmaf(v[u].z, f, o.z);
      o.w = fmaf(v[u].w, f, o.w);
    }
  }
  const float2 over = kv8_over(L);
  const int i = grow / p.G, h = kvh * p.G + grow - i * p.G;
  uint16_t* out = static_cast<uint16_t*>(p.out) + s * p.so[0] + i * p.so[1] + h * p.so[2];
  const float f[4] = {o.x * over.x * over.y, o.y * over.x * over.y, o.z * over.x * over.y, o.w * over.x * over.y};
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (d + k < p.c.D)
      out[(d + k) * p.so[3]] = p.bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(f[k])) : __half_as_ushort(__float2half_rn(f[k]));
  if (d == 0) {
    const float v = L != 0.f ? M + kLBias + log2f(L) : -INFINITY;
    if (p.lse) p.lse[(static_cast<int64_t>(s) * p.Lq + i) * p.H + h] = v * kLn2;
    if (p.lse2) p.lse2[(static_cast<int64_t>(s) * p.c.Hkv + kvh) * p.rows + grow] = v;
  }
}

// Attention weights from the stored scores: each thread owns four keys, so every
// weight is added to once, in the order of the rows.  Stored and read back, a key's
// scores cost 8 bytes a row; recomputing them would read K and multiply again.  24 x
// <= 6000 keys, 4 heads of 32 rows: 12 us (one key a thread, 18).
__global__ void __launch_bounds__(128) kv8_attention_weights_kernel(const __grid_constant__ Kv8TcParams p, int RT, float* weights,
                                                                    int64_t w0, int64_t w1, int64_t w2, int64_t width) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int kvh = blockIdx.y, s = blockIdx.z;
  const int n = static_cast<int>(min(static_cast<int64_t>(kv8_ctx(p, s)), width));
  const int pos = (blockIdx.x * 128 + threadIdx.x) * 4;
  if (pos >= n) return;
  const int64_t item = static_cast<int64_t>(s) * p.c.Hkv + kvh;
  const float* sc = p.scores + item * p.chunks * RT * p.score_ld + pos;  // a head's chunks follow one another: row r at r
  const float* ls = p.lse2 + item * p.rows;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  for (int r0 = 0; r0 < p.rows; r0 += 8) {
    float4 x[8];
    float L[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int r = min(r0 + u, p.rows - 1);
      x[u] = *reinterpret_cast<const float4*>(sc + r * p.score_ld);
      L[u] = ls[r];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float l = r0 + u < p.rows && L[u] != -INFINITY ? L[u] : INFINITY;  // rows without a key weigh nothing
      sum[0] += fast_exp2(x[u].x - l);
      sum[1] += fast_exp2(x[u].y - l);
      sum[2] += fast_exp2(x[u].z - l);
      sum[3] += fast_exp2(x[u].w - l);
    }
  }
  float* w = weights + s * w0 + kvh * w1 + pos * w2;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (pos + k < n) w[k * w2] += sum[k];
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
static bool tc_ok(const Kv8View& c, const Kv8AttnArgs& a) {
  if (a.force_generic || a.dtype == kF32 || c.D > 256 || c.P % 16 || c.group % 16) return false;
  if (c.num_blocks == 0 || c.max_blocks == 0) return false;
  if (static_cast<int64_t>(a.Lq) * a.H * c.D >= (int64_t{1} << 31)) return false;  // a sequence's query rows are counted in 32 bits
  for (const Kv8Plane& pl : c.plane) {
    if (pl.sc[3] != 1 || (reinterpret_cast<uintptr_t>(pl.code) & 15)) return false;
    for (int i = 0; i < 3; ++i)
      if (pl.sc[i] <= 0 || pl.sc[i] % 16 || pl.sc[i] >= (int64_t{1} << 40)) return false;
  }
  return true;
}
static int tc_dp(const Kv8View& c) { return c.D <= 64 ? 64 : c.D <= 128 ? 128 : 256; }
// query rows of a CTA: 8 (Kv8Few), 16 or 32 (Kv8Many), as the rows of a KV head fill
static int tc_rt(const Kv8View& c, const Kv8AttnArgs& a) {
  const int64_t rows = static_cast<int64_t>(a.H / c.Hkv) * a.Lq;
  return rows <= 8 ? 8 : rows <= 16 ? 16 : 32;
}
struct TcSizes { int N, RT, DP; int64_t places, bound, ml, o, lse2, scores, total, score_ld; };
static int64_t up16(int64_t x) { return (x + 255) / 256 * 256; }
static TcSizes tc_sizes(const Kv8View& c, const Kv8AttnArgs& a) {
  TcSizes z{};
  z.DP = tc_dp(c);
  z.RT = tc_rt(c, a);
  z.N = num_sms() * (z.DP >= 256 ? 1 : z.RT == 8 ? 3 : 2);  // CTAS of the kernel
  const int64_t rows = static_cast<int64_t>(a.H / c.Hkv) * a.Lq, all = rows * c.Hkv * c.num_seqs;
  int64_t at = 0;
  z.places = at; at += up16(8);
  z.bound = at; at += up16(static_cast<int64_t>(z.N) * 16);
  z.ml = at; at += up16(static_cast<int64_t>(z.N) * 2 * z.RT * 8);
  z.o = at; at += up16(static_cast<int64_t>(z.N) * 2 * z.RT * z.DP * 4);
  if (a.weights) {
    const int64_t w = a.weights_width < c.max_rows ? a.weights_width : c.max_rows;
    z.score_ld = (w + 15) / 16 * 16;
    z.lse2 = at; at += up16(all * 4);
    const int64_t padded = (rows + z.RT - 1) / z.RT * z.RT * c.Hkv * c.num_seqs;
    z.scores = at; at += up16(padded * z.score_ld * 4);
  }
  z.total = at + 256;
  return z;
}

int64_t kv8_attention_ws_bytes(const Kv8View& c, const Kv8AttnArgs& a) {
  if (tc_ok(c, a)) return tc_sizes(c, a).total;
  return a.weights ? static_cast<int64_t>(c.num_seqs) * a.Lq * a.H * 4 : 0;
}

static int encode_codes(CUtensorMap* map, const Kv8View& c, int w, int box_cols, int box_rows) {
  const Kv8Plane& pl = c.plane[w];
  const uint64_t dims[4] = {static_cast<uint64_t>(c.D), static_cast<uint64_t>(c.P), static_cast<uint64_t>(c.Hkv),
                            static_cast<uint64_t>(c.num_blocks)};
  const uint64_t strides[3] = {static_cast<uint64_t>(pl.sc[2]), static_cast<uint64_t>(pl.sc[1]),
                               static_cast<uint64_t>(pl.sc[0])};
  const uint32_t box[4] = {static_cast<uint32_t>(box_cols), static_cast<uint32_t>(box_rows), 1, 1};
  const uint32_t es[4] = {1, 1, 1, 1};
  return encode_tiled(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, pl.code, dims, strides, box, es,
                      box_cols == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

template <typename K, typename... A>
static int launch_dependent(K kern, dim3 grid, int threads, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  if (e == cudaSuccess) return 0;
  char buf[160];
  std::snprintf(buf, sizeof(buf), "kv8 attention: launch failed: %s", cudaGetErrorString(e));
  return set_error(3, buf);
}

template <class C, int DP, typename K>
static int launch_tc(K kern, const Kv8View& c, const Kv8AttnArgs& a, cudaStream_t st) {
  const TcSizes z = tc_sizes(c, a);
  Kv8TcParams p{};
  p.c = c;
  p.q = a.q;
  p.out = a.out;
  for (int i = 0; i < 4; ++i) { p.sq[i] = a.sq[i]; p.so[i] = a.so[i]; }
  p.context_lens = a.context_lens;
  p.lse = a.lse;
  p.bf16 = a.dtype == kBF16;
  p.q_vec = a.sq[3] == 1 && c.D % 4 == 0 && (reinterpret_cast<uintptr_t>(a.q) & 7) == 0 &&
            ((a.sq[0] | a.sq[1] | a.sq[2]) & 3) == 0;
  p.H = a.H; p.Lq = a.Lq; p.G = a.H / c.Hkv; p.rows = p.G * a.Lq;
  p.chunks = (p.rows + z.RT - 1) / z.RT;
  p.box_rows = c.P & -c.P;
  if (p.box_rows > C::CH) p.box_rows = C::CH;
  p.scale = a.softcap > 0.f ? a.scale : a.scale * kLog2e;
  p.cap2 = a.softcap * kLog2e;
  p.inv_cap = a.softcap > 0.f ? 1.f / a.softcap : 0.f;
  uint8_t* ws = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(a.workspace) + 255) & ~uintptr_t(255));
  p.places = reinterpret_cast<int64_t*>(ws + z.places);
  p.bound = reinterpret_cast<int4*>(ws + z.bound);
  p.part_ml = reinterpret_cast<float*>(ws + z.ml);
  p.part_o = reinterpret_cast<float*>(ws + z.o);
  if (a.weights) {
    p.lse2 = reinterpret_cast<float*>(ws + z.lse2);
    p.scores = reinterpret_cast<float*>(ws + z.scores);
    p.score_ld = z.score_ld;
  }
  CUtensorMap mk, mv;
  if (const int r = encode_codes(&mk, c, 0, C::ROWB, p.box_rows)) return r;
  if (const int r = encode_codes(&mv, c, 1, C::ROWB, p.box_rows)) return r;
  if (const int r = ensure_smem_attr(reinterpret_cast<const void*>(kern), C::SMEM)) return r;
  kern<<<z.N, C::THREADS, C::SMEM, st>>>(mk, mv, p);
  note_kernel("kv8_attention_tc");
  if (const int r = launch_dependent(kv8_attention_join_kernel<DP>, dim3(z.N - 1, z.RT / 4), DP, st, p, z.RT, z.N)) return r;
  if (a.weights) {
    const int64_t w = a.weights_width < c.max_rows ? a.weights_width : c.max_rows;
    return launch_dependent(kv8_attention_weights_kernel, dim3(static_cast<unsigned>((w + 511) / 512), c.Hkv, c.num_seqs),
                            128, st, p, z.RT, a.weights, a.sw[0], a.sw[1], a.sw[2], w);
  }
  return 0;
}

template <int CODE, int DP>
static int launch_rows(const Kv8View& c, const Kv8AttnArgs& a, cudaStream_t st) {
  switch (tc_rt(c, a)) {
    case 8: return launch_tc<Kv8Few<DP>, DP>(kv8_attention_few_kernel<CODE, DP>, c, a, st);
    case 16: return launch_tc<Kv8Many<DP, 2>, DP>(kv8_attention_many_kernel<CODE, DP, 2>, c, a, st);
    default: return launch_tc<Kv8Many<DP, 4>, DP>(kv8_attention_many_kernel<CODE, DP, 4>, c, a, st);
  }
}

int kv8_attention_launch(const Kv8View& c, const Kv8AttnArgs& a, cudaStream_t st) {
  if (kv8_attention_ws_bytes(c, a) > a.workspace_bytes) return set_error(4, "kv8 attention: workspace too small");
  if (!tc_ok(c, a)) return kv8_attention_generic_launch(c, a, st);
  TAK_BY_CODE(a.code_type, {
    switch (tc_dp(c)) {
      case 64: return launch_rows<CODE, 64>(c, a, st);
      case 128: return launch_rows<CODE, 128>(c, a, st);
      default: return launch_rows<CODE, 256>(c, a, st);
    }
  });
  return 0;
}

}  // namespace tak
