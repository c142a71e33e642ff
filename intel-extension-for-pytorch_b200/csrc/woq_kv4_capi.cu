// C ABI of the paged 4-bit key/value cache (declared in include/woq_b200.h): argument checks and launches.  No kernel
// code lives here.
#include <cmath>

#include "../../include/woq_b200.h"
#include "woq_internal.h"
#include "woq_kernels.h"
#include "woq_kv4_common.cuh"

namespace {

using woq::set_error;

constexpr size_t kCountersOff = 256;

#define KV4_CUDA(expr)                                                                          \
  do {                                                                                          \
    cudaError_t e__ = (expr);                                                                   \
    if (e__ != cudaSuccess)                                                                     \
      return set_error(WOQ_B200_ERR_CUDA, "%s failed: %s", #expr, cudaGetErrorString(e__));     \
  } while (0)

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check_desc(const woq_b200_kv4_desc* d) {
  if (!d) return set_error(WOQ_B200_ERR_INVALID_ARG, "the cache's description is null");
  if (d->dtype != WOQ_B200_T_BF16 && d->dtype != WOQ_B200_T_F16)
    return set_error(WOQ_B200_ERR_UNSUPPORTED, "the 4-bit cache stands for bf16 or fp16 values, got type %d", d->dtype);
  if (d->head_dim != 64 && d->head_dim != 128 && d->head_dim != 256)
    return set_error(WOQ_B200_ERR_UNSUPPORTED, "the 4-bit cache has heads of 64, 128 or 256 elements, got %d", d->head_dim);
  if ((d->group_size != 32 && d->group_size != 64 && d->group_size != 128) || d->group_size > d->head_dim)
    return set_error(WOQ_B200_ERR_UNSUPPORTED, "the 4-bit cache has groups of 32, 64 or 128 elements within a head, got %d",
                     d->group_size);
  if (d->page_size <= 0 || d->page_size % woq::kKv4Tokens || d->kv_heads < 1 || d->kv_heads > 65535 || d->num_pages < 0)
    return set_error(WOQ_B200_ERR_INVALID_ARG, "the 4-bit cache needs a page size that is a multiple of 16, 1..65535 heads "
                     "and num_pages >= 0");
  const int64_t page_bytes = static_cast<int64_t>(d->page_size / woq::kKv4Tokens) * woq::kv4_block_bytes(d->head_dim, d->group_size);
  if (d->num_pages > INT64_MAX / d->kv_heads / page_bytes)
    return set_error(WOQ_B200_ERR_INVALID_ARG, "the 4-bit cache's size passes 2^63 bytes");
  return WOQ_B200_OK;
}

int64_t block_bytes(const woq_b200_kv4_desc* d) { return woq::kv4_block_bytes(d->head_dim, d->group_size); }

int check_rows(const char* what, const void* p, int64_t tok, int64_t head) {
  if (!p) return set_error(WOQ_B200_ERR_INVALID_ARG, "%s is null", what);
  if (!aligned16(p) || tok % 8 || head % 8)
    return set_error(WOQ_B200_ERR_INVALID_ARG, "%s must be 16-byte aligned with strides that are multiples of 8 elements", what);
  return WOQ_B200_OK;
}

int num_sms(int* out) {
  int dev = 0;
  KV4_CUDA(cudaGetDevice(&dev));
  KV4_CUDA(cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, dev));
  return WOQ_B200_OK;
}

size_t partials_off() { return woq_b200_workspace_header_bytes(); }

}  // namespace

extern "C" {

size_t woq_b200_kv4_bytes(const woq_b200_kv4_desc* d) {
  if (check_desc(d) != WOQ_B200_OK) return 0;
  return static_cast<size_t>(d->num_pages) * d->kv_heads * (d->page_size / woq::kKv4Tokens) * block_bytes(d);
}

int woq_b200_kv4_append(const woq_b200_kv4_desc* d, void* cache, const void* q, int64_t q_tok, int64_t q_head,
                        int32_t q_heads, const void* k, int64_t k_tok, int64_t k_head, const void* v, int64_t v_tok,
                        int64_t v_head, const int64_t* slots, const int64_t* positions, const float* cos_sin,
                        int64_t max_pos, int32_t rot, int32_t interleaved, int64_t tokens, void* q_out, void* stream) {
  if (int rc = check_desc(d)) return rc;
  if (tokens < 0 || tokens > INT32_MAX || q_heads < 0 || q_heads > 65535)
    return set_error(WOQ_B200_ERR_INVALID_ARG, "0 <= tokens < 2^31 and 0 <= q_heads < 2^16");
  if (rot < 0 || rot > d->head_dim || rot % 16)
    return set_error(WOQ_B200_ERR_UNSUPPORTED, "the rotated part of a head is a multiple of 16 elements, at most all %d, got %d",
                     d->head_dim, rot);
  if (tokens == 0) return WOQ_B200_OK;
  if (!slots || (d->num_pages > 0 && !cache)) return set_error(WOQ_B200_ERR_INVALID_ARG, "cache and slots must be non-null");
  if (!aligned16(cache)) return set_error(WOQ_B200_ERR_INVALID_ARG, "the cache must be 16-byte aligned");
  if (rot > 0 && (!positions || !cos_sin || max_pos < 1 || !aligned16(cos_sin)))
    return set_error(WOQ_B200_ERR_INVALID_ARG, "a rotation needs positions and a 16-byte aligned table of cosines and sines");
  if (q_heads > 0) {
    if (int rc = check_rows("q", q, q_tok, q_head)) return rc;
    if (!q_out || !aligned16(q_out)) return set_error(WOQ_B200_ERR_INVALID_ARG, "q_out must be non-null and 16-byte aligned");
  }
  if (int rc = check_rows("k", k, k_tok, k_head)) return rc;
  if (int rc = check_rows("v", v, v_tok, v_head)) return rc;
  woq::Kv4AppendParams p{};
  p.q = static_cast<const uint16_t*>(q);
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.q_out = static_cast<uint16_t*>(q_out);
  p.cache = static_cast<uint8_t*>(cache);
  p.slots = slots;
  p.positions = rot > 0 ? positions : nullptr;
  p.cos_sin = cos_sin;
  p.q_tok = q_tok;
  p.q_head = q_head;
  p.k_tok = k_tok;
  p.k_head = k_head;
  p.v_tok = v_tok;
  p.v_head = v_head;
  p.max_pos = max_pos;
  p.num_slots = d->num_pages * d->page_size;
  p.q_heads = q_heads;
  p.kv_heads = d->kv_heads;
  p.page_blocks = d->page_size / woq::kKv4Tokens;
  p.rot = rot;
  p.interleaved = interleaved != 0;
  KV4_CUDA(woq::launch_kv4_append(p, d->dtype == WOQ_B200_T_F16, d->head_dim, d->group_size, tokens,
                                  static_cast<cudaStream_t>(stream)));
  return WOQ_B200_OK;
}

int woq_b200_kv4_read(const woq_b200_kv4_desc* d, const void* cache, const int64_t* slots, int64_t tokens, void* k,
                      void* v, void* stream) {
  if (int rc = check_desc(d)) return rc;
  if (tokens < 0 || tokens > INT32_MAX) return set_error(WOQ_B200_ERR_INVALID_ARG, "0 <= tokens < 2^31");
  if (tokens == 0) return WOQ_B200_OK;
  if (!slots || (d->num_pages > 0 && !cache)) return set_error(WOQ_B200_ERR_INVALID_ARG, "cache and slots must be non-null");
  if (!aligned16(cache)) return set_error(WOQ_B200_ERR_INVALID_ARG, "the cache must be 16-byte aligned");
  if (int rc = check_rows("k", k, 0, 0)) return rc;
  if (int rc = check_rows("v", v, 0, 0)) return rc;
  woq::Kv4ReadParams p{};
  p.cache = static_cast<const uint8_t*>(cache);
  p.slots = slots;
  p.k = static_cast<uint16_t*>(k);
  p.v = static_cast<uint16_t*>(v);
  p.tokens = tokens;
  p.num_slots = d->num_pages * d->page_size;
  p.kv_heads = d->kv_heads;
  p.page_blocks = d->page_size / woq::kKv4Tokens;
  KV4_CUDA(woq::launch_kv4_read(p, d->dtype == WOQ_B200_T_F16, d->head_dim, d->group_size, static_cast<cudaStream_t>(stream)));
  return WOQ_B200_OK;
}

size_t woq_b200_kv4_attention_workspace_bytes(const woq_b200_kv4_desc* d, int64_t batch, int64_t tokens, int32_t q_heads) {
  if (check_desc(d) != WOQ_B200_OK || batch < 0 || batch > INT32_MAX || tokens < 0 || tokens > INT32_MAX || q_heads < 1 ||
      q_heads % d->kv_heads)
    return 0;
  int sms = 0;
  if (num_sms(&sms) != WOQ_B200_OK) return 0;
  if (batch == 0 || tokens == 0) return partials_off();
  return partials_off() + woq::kv4_attend_partial_bytes_up_to(tokens, q_heads / d->kv_heads, d->kv_heads, d->head_dim, sms);
}

int woq_b200_kv4_attention(const woq_b200_kv4_desc* d, const void* cache, const void* q, int64_t q_tok, int64_t q_head,
                           int32_t q_heads, const int32_t* block_table, int64_t table_ld, int64_t max_pages,
                           const int32_t* seq_lens, const int32_t* query_starts, int64_t batch, int64_t tokens, float scale,
                           int32_t causal, void* out, int64_t o_tok, int64_t o_head, void* workspace,
                           size_t workspace_bytes, void* stream) {
  if (int rc = check_desc(d)) return rc;
  if (batch < 0 || batch > INT32_MAX || tokens < 0 || tokens > INT32_MAX || max_pages < 0)
    return set_error(WOQ_B200_ERR_INVALID_ARG, "0 <= batch, tokens < 2^31 and max_pages >= 0");
  if (q_heads < 1 || q_heads % d->kv_heads)
    return set_error(WOQ_B200_ERR_INVALID_ARG, "the number of query heads (%d) must be a multiple of the cache's %d", q_heads,
                     d->kv_heads);
  if (!query_starts && batch != tokens)
    return set_error(WOQ_B200_ERR_INVALID_ARG, "without query_starts every sequence has one query row: %lld rows for %lld "
                     "sequences", (long long)tokens, (long long)batch);
  if (!(std::fabs(scale) < 1e18f)) return set_error(WOQ_B200_ERR_INVALID_ARG, "the scale must be a number below 1e18");
  if (tokens == 0 || batch == 0) return WOQ_B200_OK;
  // (kernels number keys in 31 bits, up to three tiles of 128 and a warp of blocks behind the last one)
  if (max_pages > 0 && (INT32_MAX - 1023) / max_pages < d->page_size)
    return set_error(WOQ_B200_ERR_UNSUPPORTED, "a block table of %lld pages of %d tokens passes 2^31 - 1024 tokens",
                     (long long)max_pages, d->page_size);
  const int heads = q_heads / d->kv_heads;
  // tiles of eight query rows, and their units of 32 keys (whose number in a CTA's share has 31 bits)
  const double items = (static_cast<double>(tokens) * heads / 8 + static_cast<double>(batch)) * d->kv_heads;
  if (tokens > (INT32_MAX - 1023) / heads || items > 2e9 || items * (20 + max_pages * (d->page_size / 32.0)) > 3e11)
    return set_error(WOQ_B200_ERR_UNSUPPORTED, "too many query rows and cached tokens for one call");
  if (!seq_lens || (max_pages > 0 && !block_table) || !workspace || (d->num_pages > 0 && !cache))
    return set_error(WOQ_B200_ERR_INVALID_ARG, "cache, block_table, seq_lens and workspace must be non-null");
  if (!aligned16(cache) || !aligned16(workspace))
    return set_error(WOQ_B200_ERR_INVALID_ARG, "cache and workspace must be 16-byte aligned");
  if (table_ld < max_pages) return set_error(WOQ_B200_ERR_INVALID_ARG, "table_ld is smaller than max_pages");
  if (int rc = check_rows("q", q, q_tok, q_head)) return rc;
  if (int rc = check_rows("out", out, o_tok, o_head)) return rc;
  int sms = 0;
  if (int rc = num_sms(&sms)) return rc;
  const size_t need = partials_off() + woq::kv4_attend_partial_bytes(static_cast<int>(batch), tokens, heads, d->kv_heads, d->head_dim, sms);
  if (workspace_bytes < need)
    return set_error(WOQ_B200_ERR_WORKSPACE, "workspace has %zu bytes, need %zu", workspace_bytes, need);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  woq::Kv4AttendParams p{};
  p.q = static_cast<const uint16_t*>(q);
  p.out = static_cast<uint16_t*>(out);
  p.cache = static_cast<const uint8_t*>(cache);
  p.table = block_table;
  p.lens = seq_lens;
  p.starts = query_starts;
  p.status = reinterpret_cast<int*>(ws);
  p.counters = reinterpret_cast<uint32_t*>(ws + kCountersOff);
  p.partials = reinterpret_cast<float*>(ws + partials_off());
  p.q_tok = q_tok;
  p.q_head = q_head;
  p.o_tok = o_tok;
  p.o_head = o_head;
  p.table_ld = table_ld;
  p.num_pages = d->num_pages;
  p.scale = scale * 1.4426950408889634f;  // log2 e: the kernel's exponentials are powers of two
  p.batch = static_cast<int>(batch);
  p.tokens = static_cast<int>(tokens);
  p.kv_heads = d->kv_heads;
  p.heads = heads;
  p.page_blocks = d->page_size / woq::kKv4Tokens;
  p.max_blocks = static_cast<int>(max_pages * p.page_blocks);
  p.causal = causal != 0;
  KV4_CUDA(woq::launch_kv4_attend(p, d->dtype == WOQ_B200_T_F16, d->head_dim, d->group_size, sms,
                                  static_cast<cudaStream_t>(stream)));
  return WOQ_B200_OK;
}

}  // extern "C"
