// extern "C" entry points of the rotary positions and the 8-bit KV cache
// (include/tak_attention.h): argument checks and dispatch.
#include "kv8.cuh"

using namespace tak;

#define TAK_REQUIRE(cond, msg) \
  do {                         \
    if (!(cond)) return set_error(1, msg); \
  } while (0)

constexpr int64_t kMaxInt = 0x7fffffff;
// Rows of a sequence: positions are 32-bit, and the kernels look up to a step of
// thousands of rows past the last one.
constexpr int64_t kMaxRows = kMaxInt - 0xffff;
// Caps between these have fp32 reciprocals, and cap * log2(e) is finite.  Scores are
// far below 2^126, where the cap is the identity: a larger one, infinity too, is none.
constexpr float kMinCap = 1.17549435082228751e-38f;  // 2^-126
constexpr float kMaxCap = 8.50705917302346159e37f;   // 2^126

static void strides_to(int64_t* dst, const int64_t* src, int n) {
  for (int i = 0; i < n; ++i) dst[i] = src[i];
}

// Checks a cache description and fills the kernels' view of it.
static int make_view(Kv8View* out, const tak_kv8_cache* c) {
  TAK_REQUIRE(c, "kv8: null cache description");
  TAK_REQUIRE(c->code_type == TAK_KV8_INT8 || c->code_type == TAK_KV8_E4M3, "kv8: unknown code type");
  TAK_REQUIRE(c->num_kv_heads > 0 && c->num_kv_heads <= 65535, "kv8: num_kv_heads must be in [1, 65535]");
  TAK_REQUIRE(c->head_dim > 0 && c->head_dim <= 640, "kv8: head_dim must be in [1, 640]");
  TAK_REQUIRE(c->block_size > 0 && c->block_size <= 65536, "kv8: block_size must be in [1, 65536]");
  TAK_REQUIRE(c->group > 0 && c->group <= 256 && c->block_size % c->group == 0,
              "kv8: group must divide block_size and be in [1, 256]");
  TAK_REQUIRE(c->num_seqs >= 0 && c->num_seqs <= 65535, "kv8: num_seqs must be in [0, 65535]");
  TAK_REQUIRE(c->num_blocks >= 0 && c->num_blocks <= kMaxInt, "kv8: num_blocks must be in [0, 2^31)");
  TAK_REQUIRE(c->max_blocks >= 0 && c->max_blocks <= kMaxRows / c->block_size,
              "kv8: max_blocks * block_size must be at most 2^31 - 2^16");
  Kv8View v{};
  v.Hkv = static_cast<int>(c->num_kv_heads);
  v.P = static_cast<int>(c->block_size);
  v.D = static_cast<int>(c->head_dim);
  v.group = static_cast<int>(c->group);
  v.num_seqs = static_cast<int>(c->num_seqs);
  v.max_blocks = static_cast<int>(c->max_blocks);
  v.num_blocks = c->num_blocks;
  v.max_rows = c->max_blocks * c->block_size;
  v.by_P = kv8_div_by(static_cast<uint32_t>(v.P));
  v.by_group = kv8_div_by(static_cast<uint32_t>(v.group));
  if (v.num_blocks > 0) TAK_REQUIRE(c->k_cache && c->v_cache && c->k_scale && c->v_scale, "kv8: null cache pointer");
  if (v.num_seqs > 0 && v.max_blocks > 0) TAK_REQUIRE(c->block_tables, "kv8: null block table");
  v.plane[0].code = static_cast<uint8_t*>(c->k_cache);
  v.plane[1].code = static_cast<uint8_t*>(c->v_cache);
  v.plane[0].scale = c->k_scale;
  v.plane[1].scale = c->v_scale;
  strides_to(v.plane[0].sc, c->k_strides, 4);
  strides_to(v.plane[1].sc, c->v_strides, 4);
  strides_to(v.plane[0].ss, c->k_scale_strides, 3);
  strides_to(v.plane[1].ss, c->v_scale_strides, 3);
  v.block_tables = c->block_tables;
  strides_to(v.sbt, c->bt_strides, 2);
  *out = v;
  return 0;
}

extern "C" {

int tak_rotary_nd(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                  const int32_t* positions, const int64_t* pos_strides, const float* inv_freq,
                  const int32_t* sections, int64_t num_axes, void* q_out, const int64_t* q_out_strides, void* k_out,
                  const int64_t* k_out_strides, int64_t total_tokens, int64_t num_q_heads, int64_t num_kv_heads,
                  int64_t head_dim, int64_t rot_dim, int interleaved, int inverse, int dtype, void* stream) {
  note_kernel("");
  TAK_REQUIRE(dtype >= 0 && dtype <= 2, "rotary: unknown dtype");
  TAK_REQUIRE(total_tokens >= 0 && total_tokens <= kMaxInt, "rotary: total_tokens must be in [0, 2^31)");
  TAK_REQUIRE(num_q_heads >= 0 && num_kv_heads >= 0 && num_q_heads + num_kv_heads <= 65535,
              "rotary: the numbers of heads must be in [0, 65535]");
  TAK_REQUIRE(head_dim > 0 && head_dim <= 1024, "rotary: head_dim must be in [1, 1024]");
  TAK_REQUIRE(rot_dim >= 0 && rot_dim <= head_dim && rot_dim % 2 == 0,
              "rotary: rot_dim must be even and at most head_dim");
  TAK_REQUIRE(num_axes >= 1 && num_axes <= 8 && sections, "rotary: 1 to 8 axes");
  RotaryArgs a{};
  int64_t end = 0;
  for (int i = 0; i < num_axes; ++i) {
    TAK_REQUIRE(sections[i] >= 0, "rotary: negative section");
    end += sections[i];
    a.section_end[i] = static_cast<int>(end);
  }
  TAK_REQUIRE(end == rot_dim / 2, "rotary: the sections must add up to rot_dim / 2");
  if (total_tokens == 0 || num_q_heads + num_kv_heads == 0) return 0;
  TAK_REQUIRE(num_q_heads == 0 || (q && q_out && q_strides && q_out_strides), "rotary: null q");
  TAK_REQUIRE(num_kv_heads == 0 || (k && k_out && k_strides && k_out_strides), "rotary: null k");
  TAK_REQUIRE(rot_dim == 0 || (positions && pos_strides && inv_freq), "rotary: null positions or inv_freq");
  a.q = q; a.k = k; a.q_out = q_out; a.k_out = k_out;
  if (num_q_heads) { strides_to(a.sq, q_strides, 3); strides_to(a.sqo, q_out_strides, 3); }
  if (num_kv_heads) { strides_to(a.sk, k_strides, 3); strides_to(a.sko, k_out_strides, 3); }
  a.positions = positions;
  if (rot_dim) strides_to(a.sp, pos_strides, 2);
  a.inv_freq = inv_freq;
  a.axes = static_cast<int>(num_axes);
  a.total_tokens = static_cast<int>(total_tokens);
  a.num_q_heads = static_cast<int>(num_q_heads);
  a.num_kv_heads = static_cast<int>(num_kv_heads);
  a.head_dim = static_cast<int>(head_dim);
  a.rot_dim = static_cast<int>(rot_dim);
  a.interleaved = interleaved;
  a.inverse = inverse;
  a.dtype = dtype;
  const int r = rotary_nd_launch(a, static_cast<cudaStream_t>(stream));
  return r ? r : check_launch("rotary");
}

int tak_kv8_write(const tak_kv8_cache* cache, const void* k, const int64_t* k_strides, const void* v,
                  const int64_t* v_strides, const int32_t* start_lens, const int32_t* cu_seqlens,
                  int64_t total_tokens, int dtype, void* stream) {
  note_kernel("");
  Kv8View c;
  if (const int r = make_view(&c, cache)) return r;
  TAK_REQUIRE(dtype >= 0 && dtype <= 2, "kv8 write: unknown dtype");
  TAK_REQUIRE(total_tokens >= 0 && total_tokens <= kMaxInt, "kv8 write: total_tokens must be in [0, 2^31)");
  TAK_REQUIRE(cu_seqlens || total_tokens == c.num_seqs, "kv8 write: one row per sequence without cu_seqlens");
  if (total_tokens == 0 || c.num_seqs == 0) return 0;
  TAK_REQUIRE(k && v && k_strides && v_strides && start_lens, "kv8 write: null pointer");
  const int r = kv8_write_launch(c, static_cast<int>(cache->code_type), k, k_strides, v, v_strides, start_lens,
                                 cu_seqlens, total_tokens, dtype, static_cast<cudaStream_t>(stream));
  return r ? r : check_launch("kv8 write");
}

int tak_kv8_read(const tak_kv8_cache* cache, const int32_t* cu_seqlens, const int32_t* start_lens,
                 int64_t total_tokens, void* k, const int64_t* k_strides, void* v, const int64_t* v_strides,
                 int dtype, void* stream) {
  note_kernel("");
  Kv8View c;
  if (const int r = make_view(&c, cache)) return r;
  TAK_REQUIRE(dtype >= 0 && dtype <= 2, "kv8 read: unknown dtype");
  TAK_REQUIRE(total_tokens >= 0 && total_tokens <= kMaxInt, "kv8 read: total_tokens must be in [0, 2^31)");
  if (total_tokens == 0) return 0;
  TAK_REQUIRE(c.num_seqs > 0, "kv8 read: rows asked for of no sequence");
  TAK_REQUIRE(k && v && k_strides && v_strides && cu_seqlens, "kv8 read: null pointer");
  const int r = kv8_read_launch(c, static_cast<int>(cache->code_type), cu_seqlens, start_lens, total_tokens, k,
                                k_strides, v, v_strides, dtype, static_cast<cudaStream_t>(stream));
  return r ? r : check_launch("kv8 read");
}

static int make_attn(Kv8AttnArgs* out, const Kv8View& c, int64_t num_q_heads, int64_t num_queries, int64_t width,
                     int code_type, int dtype) {
  TAK_REQUIRE(dtype >= 0 && dtype <= 2, "kv8 attention: unknown dtype");
  TAK_REQUIRE(width >= 0 && width <= kMaxInt, "kv8 attention: weights_width must be in [0, 2^31)");
  TAK_REQUIRE(num_q_heads > 0 && num_q_heads <= 65535 && num_q_heads % c.Hkv == 0,
              "kv8 attention: num_q_heads must be a multiple of num_kv_heads, at most 65535");
  TAK_REQUIRE(num_queries >= 0 && num_queries <= 65535, "kv8 attention: num_queries must be in [0, 65535]");
  Kv8AttnArgs a{};
  a.H = static_cast<int>(num_q_heads);
  a.Lq = static_cast<int>(num_queries);
  a.weights_width = width;
  a.code_type = code_type;
  a.dtype = dtype;
  a.force_generic = kernel_path() == 1;
  *out = a;
  return 0;
}

int64_t tak_kv8_attention_workspace_size(const tak_kv8_cache* cache, int64_t num_q_heads, int64_t num_queries,
                                         int64_t weights_width, int dtype) {
  Kv8View c;
  Kv8AttnArgs a;
  if (make_view(&c, cache) || make_attn(&a, c, num_q_heads, num_queries, weights_width,
                                        static_cast<int>(cache->code_type), dtype))
    return -1;
  static float dummy;
  a.weights = weights_width > 0 ? &dummy : nullptr;
  return kv8_attention_ws_bytes(c, a);
}

int tak_kv8_attention(const tak_kv8_cache* cache, const void* q, const int64_t* q_strides,
                      const int32_t* context_lens, void* out, const int64_t* out_strides, float* lse,
                      float* weights, const int64_t* weights_strides, int64_t weights_width, int64_t num_q_heads,
                      int64_t num_queries, float scale, float softcap, int dtype, void* workspace,
                      int64_t workspace_bytes, void* stream) {
  note_kernel("");
  Kv8View c;
  if (const int r = make_view(&c, cache)) return r;
  TAK_REQUIRE(softcap == 0.f || softcap >= kMinCap, "kv8 attention: softcap must be 0 (none) or at least 2^-126");
  Kv8AttnArgs a;
  if (const int r = make_attn(&a, c, num_q_heads, num_queries, weights_width, static_cast<int>(cache->code_type), dtype))
    return r;
  if (c.num_seqs == 0 || num_queries == 0) return 0;
  TAK_REQUIRE(q && q_strides && out && out_strides && context_lens, "kv8 attention: null pointer");
  TAK_REQUIRE(!weights || weights_strides, "kv8 attention: null weights strides");
  a.q = q; strides_to(a.sq, q_strides, 4);
  a.out = out; strides_to(a.so, out_strides, 4);
  a.context_lens = context_lens;
  a.lse = lse;
  a.weights = weights_width > 0 ? weights : nullptr;
  if (weights) strides_to(a.sw, weights_strides, 3);
  a.scale = scale;
  a.softcap = softcap <= kMaxCap ? softcap : 0.f;
  a.workspace = workspace;
  a.workspace_bytes = workspace ? workspace_bytes : 0;
  const int r = kv8_attention_launch(c, a, static_cast<cudaStream_t>(stream));
  return r ? r : check_launch("kv8 attention");
}

int tak_kv8_evict(const tak_kv8_cache* cache, const int32_t* context_lens, float* weights,
                  const int64_t* weights_strides, int64_t weights_width, int64_t budget, int64_t recent,
                  int32_t* kept, int32_t* new_lens, void* stream) {
  note_kernel("");
  Kv8View c;
  if (const int r = make_view(&c, cache)) return r;
  TAK_REQUIRE(weights_width >= 0 && weights_width <= kMaxInt, "kv8 evict: weights_width must be in [0, 2^31)");
  TAK_REQUIRE(budget >= 1 && budget <= kMaxInt, "kv8 evict: budget must be in [1, 2^31)");
  TAK_REQUIRE(recent >= 0 && recent <= budget, "kv8 evict: recent must be in [0, budget]");
  if (c.num_seqs == 0) return 0;
  TAK_REQUIRE(context_lens && kept && new_lens, "kv8 evict: null pointer");
  TAK_REQUIRE(weights_width == 0 || (weights && weights_strides), "kv8 evict: null weights");
  int64_t zero[3] = {0, 0, 0};
  const int r = kv8_evict_launch(c, static_cast<int>(cache->code_type), context_lens, weights,
                                 weights_strides ? weights_strides : zero, weights_width, budget, recent, kept,
                                 new_lens, static_cast<cudaStream_t>(stream));
  return r ? r : check_launch("kv8 evict");
}

}  // extern "C"
