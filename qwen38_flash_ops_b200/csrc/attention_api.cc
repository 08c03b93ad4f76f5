// The C ABI of heads, their cache and attention: checks of arguments, and the calls into their kernels.
#include <atomic>
#include <climits>
#include <cmath>
#include <cstdlib>
#include <cstring>
#include <exception>
#include <stdexcept>
#include <string>

#include "qfg_internal.h"

struct qfg_qk_norm_rope {
  int dim = 0, n_pairs = 0, axes = 1;
  bool interleaved = false;
  float rotary_scale = 1.f, eps = 0.f, weight_offset = 0.f;
  qfg::RotaryPair* pairs = nullptr;  // on the device
  int device = -1;
};

namespace {

int Refuse(const char* name, const std::string& why) { return qfg::SetLastError(QFG_INVALID_ARGUMENT, (std::string(name) + ": " + why).c_str()); }
int Launched(const char* name, cudaError_t err) {
  return err == cudaSuccess ? QFG_OK : qfg::SetLastError(QFG_FAIL, (std::string(name) + ": " + cudaGetErrorString(err)).c_str());
}
size_t BytesOf(int dtype) { return dtype == QFG_FLOAT ? 4 : dtype == QFG_BFLOAT16 || dtype == QFG_FLOAT16 ? 2 : 0; }
bool On(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
bool Dim(int64_t d) { return d == 64 || d == 128 || d == 256; }
constexpr int64_t kMostHeads = 4096;

// A cache's description; false with the reason set.
int CheckCache(const char* name, const qfg_kv_cache* c, qfg::KvCacheView* v) {
  if (c == nullptr) return Refuse(name, "null cache");
  if (c->dtype != QFG_UINT8 && c->dtype != QFG_FLOAT8E4M3FN) return Refuse(name, "a cache holds UINT8 (block-16 NVFP4) or FP8 E4M3FN");
  if (!Dim(c->head_dim)) return Refuse(name, "heads must have 64, 128 or 256 channels");
  if (c->pages < 1 || c->kv_heads < 1 || c->kv_heads > kMostHeads) return Refuse(name, "a cache has at least one page and 1 to 4096 heads");
  if (c->page < 32 || c->page > 65536 || c->page % 32 != 0) return Refuse(name, "the tokens of a page must be a multiple of 32, up to 65536");
  if (c->pages > LLONG_MAX / (static_cast<int64_t>(c->kv_heads) * c->page * c->head_dim)) return Refuse(name, "the cache is too large");
  if (c->pages > INT_MAX) return Refuse(name, "a cache has at most 2147483647 pages");
  if (c->k == nullptr || c->v == nullptr || c->k_scale == nullptr || c->v_scale == nullptr) return Refuse(name, "null cache");
  if (!On(c->k, 16) || !On(c->v, 16) || !On(c->k_scale, 16) || !On(c->v_scale, 16)) return Refuse(name, "the cache's tensors must begin on 16 bytes");
  const bool fp4 = c->dtype == QFG_UINT8;
  if (fp4 && !(c->k_unit >= 1e-18f && c->k_unit <= 1e18f && c->v_unit >= 1e-18f && c->v_unit <= 1e18f)) return Refuse(name, "the units must lie between 1e-18 and 1e18");
  v->k = static_cast<uint8_t*>(c->k);
  v->v = static_cast<uint8_t*>(c->v);
  v->k_scale = c->k_scale;
  v->v_scale = c->v_scale;
  v->pages = c->pages;
  v->heads = static_cast<int>(c->kv_heads);
  v->page = static_cast<int>(c->page);
  v->dim = static_cast<int>(c->head_dim);
  v->fp4 = fp4;
  v->k_unit = fp4 ? c->k_unit : 1.f;
  v->v_unit = fp4 ? c->v_unit : 1.f;
  return QFG_OK;
}

// rows of heads [tokens][heads][dim], tokens ld elements apart
int CheckHeads(const char* name, const char* what, const void* x, int64_t ld, int64_t heads, int64_t dim, size_t elem) {
  if (x == nullptr) return Refuse(name, std::string("null ") + what);
  if (heads < 1 || heads > kMostHeads) return Refuse(name, std::string(what) + " must have 1 to 4096 heads");
  if (ld < heads * dim) return Refuse(name, std::string("the rows of ") + what + " overlap");
  if (!On(x, elem)) return Refuse(name, std::string(what) + " is misaligned");
  return QFG_OK;
}
bool Scale(float s) { return s > 0.f && s <= 1e18f; }
std::atomic<bool> g_prompt_give_up{false};  // qfg_prompt_attention_set_option

}  // namespace

#define QFG_CHECK(call)              \
  do {                               \
    const int qfg_code = (call);     \
    if (qfg_code != QFG_OK) return qfg_code; \
  } while (0)

int qfg_qk_norm_rope_create(const double* inv_freq, const int32_t* axis, int n_pairs, int head_dim, int interleaved, float rotary_scale, float eps,
                            float weight_offset, qfg_qk_norm_rope** out) {
  const char* const name = "QkNormRope";
  if (out == nullptr) return Refuse(name, "null handle pointer");
  *out = nullptr;
  if (!Dim(head_dim)) return Refuse(name, "heads must have 64, 128 or 256 channels");
  if (n_pairs < 0 || n_pairs % 16 != 0 || 2 * n_pairs > head_dim) return Refuse(name, "the rotated channels must be a multiple of 32, at most the head's");
  if (n_pairs > 0 && inv_freq == nullptr) return Refuse(name, "null frequencies");
  if (!(eps >= 0.f) || !std::isfinite(rotary_scale) || !std::isfinite(weight_offset)) return Refuse(name, "eps must not be negative, and every factor finite");
  qfg_qk_norm_rope* op = nullptr;
  try {
    op = new qfg_qk_norm_rope();
    op->dim = head_dim;
    op->n_pairs = n_pairs;
    op->interleaved = interleaved != 0;
    op->rotary_scale = rotary_scale;
    op->eps = eps;
    op->weight_offset = weight_offset;
    std::string pairs(static_cast<size_t>(n_pairs) * sizeof(qfg::RotaryPair), '\0');
    for (int i = 0; i < n_pairs; ++i) {
      const int a = axis != nullptr ? axis[i] : 0;
      if (!std::isfinite(inv_freq[i])) throw std::invalid_argument("the frequencies must be finite");
      if (a < 0 || a > 7) throw std::invalid_argument("a pair's axis must be 0 to 7");
      // radians a position, as a fraction of a turn
      const long double turns = static_cast<long double>(inv_freq[i]) / 6.283185307179586476925286766559L, part = turns - std::floor(turns);
      const long double of = std::ldexp(part, 64);
      qfg::RotaryPair& p = reinterpret_cast<qfg::RotaryPair*>(&pairs[0])[i];
      p.turns = of >= 18446744073709551615.0L ? 0ull : static_cast<unsigned long long>(of);
      p.axis = a;
      op->axes = a + 1 > op->axes ? a + 1 : op->axes;
    }
    cudaError_t err = cudaGetDevice(&op->device);
    if (err == cudaSuccess && n_pairs > 0) err = cudaMalloc(reinterpret_cast<void**>(&op->pairs), pairs.size());
    if (err == cudaSuccess && n_pairs > 0) err = cudaMemcpy(op->pairs, pairs.data(), pairs.size(), cudaMemcpyHostToDevice);
    // a copy from pageable memory may return ahead of its last part, and the node may be used on a stream that does not wait for the default one
    if (err == cudaSuccess && n_pairs > 0) err = cudaStreamSynchronize(nullptr);
    if (err != cudaSuccess) throw std::runtime_error(cudaGetErrorString(err));
  } catch (const std::invalid_argument& e) {
    delete op;
    return Refuse(name, e.what());
  } catch (const std::exception& e) {
    if (op != nullptr) cudaFree(op->pairs);
    delete op;
    return qfg::SetLastError(QFG_FAIL, (std::string(name) + ": " + e.what()).c_str());
  }
  *out = op;
  return QFG_OK;
}

void qfg_qk_norm_rope_destroy(qfg_qk_norm_rope* op) {
  if (op == nullptr) return;
  cudaFree(op->pairs);
  delete op;
}

int qfg_qk_norm_rope_compute(const qfg_qk_norm_rope* op, int dtype, const void* q, int64_t ldq, int64_t q_heads, const void* k, int64_t ldk, int64_t kv_heads,
                             const void* v, int64_t ldv, const void* positions, int position_bytes, int64_t ld_positions, int64_t axes, const void* q_weight,
                             const void* k_weight, int weight_dtype, int64_t tokens, void* q_out, void* k_out, const qfg_kv_cache* cache, const int64_t* slots,
                             void* stream) {
  const char* const name = "QkNormRope";
  if (op == nullptr) return Refuse(name, "null node");
  const size_t elem = BytesOf(dtype);
  if (elem == 0) return Refuse(name, "heads must be BF16/FP16/FP32");
  if (tokens < 0 || tokens > INT_MAX / 2) return Refuse(name, "bad number of tokens");
  qfg::HeadsCall c;
  if (cache != nullptr) {
    QFG_CHECK(CheckCache(name, cache, &c.cache));
    if (c.cache.dim != op->dim || c.cache.heads != kv_heads) return Refuse(name, "the cache has other heads");
  }
  if (tokens == 0) return QFG_OK;
  int device = -1;
  if (cudaGetDevice(&device) != cudaSuccess || device != op->device) return Refuse(name, "the node was made on another device");
  QFG_CHECK(CheckHeads(name, "q", q, ldq, q_heads, op->dim, elem));
  QFG_CHECK(CheckHeads(name, "k", k, ldk, kv_heads, op->dim, elem));
  if (cache != nullptr) QFG_CHECK(CheckHeads(name, "v", v, ldv, kv_heads, op->dim, elem));
  if (op->n_pairs > 0) {
    if (positions == nullptr || (position_bytes != 4 && position_bytes != 8) || !On(positions, static_cast<size_t>(position_bytes)))
      return Refuse(name, "positions must be 32-bit or 64-bit integers");
    if (axes != op->axes || (axes > 1 && ld_positions < tokens)) return Refuse(name, "positions must be [" + (op->axes > 1 ? std::to_string(op->axes) + ", " : std::string()) + std::to_string(tokens) + "]");
  }
  if ((q_weight != nullptr || k_weight != nullptr) && weight_dtype != dtype && weight_dtype != QFG_FLOAT)
    return Refuse(name, "the weights must have the type of the heads, or FP32");
  if (!On(q_weight, BytesOf(weight_dtype) ? BytesOf(weight_dtype) : 1) || !On(k_weight, BytesOf(weight_dtype) ? BytesOf(weight_dtype) : 1))
    return Refuse(name, "a weight is misaligned");
  if (q_out == nullptr || !On(q_out, 16) || !On(k_out, 16)) return Refuse(name, "the outputs must begin on 16 bytes");
  if (cache != nullptr ? slots == nullptr || !On(slots, 8) : k_out == nullptr) return Refuse(name, cache != nullptr ? "no slots" : "no output for the keys");
  c.dtype = dtype;
  c.dim = op->dim;
  c.q = q;
  c.ldq = ldq;
  c.q_heads = static_cast<int>(q_heads);
  c.k = k;
  c.ldk = ldk;
  c.kv_heads = static_cast<int>(kv_heads);
  c.v = cache != nullptr ? v : nullptr;
  c.ldv = ldv;
  c.q_weight = q_weight;
  c.k_weight = k_weight;
  c.weight_dtype = weight_dtype;
  c.weight_offset = op->weight_offset;
  c.eps = op->eps;
  c.pairs = op->pairs;
  c.n_pairs = op->n_pairs;
  c.interleaved = op->interleaved;
  c.rotary_scale = op->rotary_scale;
  c.positions = positions;
  c.positions_64 = position_bytes == 8;
  c.ld_positions = ld_positions;
  c.tokens = tokens;
  c.q_out = q_out;
  c.k_out = k_out;
  c.slots = cache != nullptr ? slots : nullptr;
  return Launched(name, qfg::LaunchHeadRows(c, static_cast<cudaStream_t>(stream)));
}

int qfg_cache_write(int dtype, const void* k, int64_t ldk, const void* v, int64_t ldv, int64_t tokens, const qfg_kv_cache* cache, const int64_t* slots, void* stream) {
  const char* const name = "CacheWrite";
  qfg::HeadsCall c;
  QFG_CHECK(CheckCache(name, cache, &c.cache));
  const size_t elem = BytesOf(dtype);
  if (elem == 0) return Refuse(name, "keys and values must be BF16/FP16/FP32");
  if (tokens < 0 || tokens > INT_MAX / 2) return Refuse(name, "bad number of tokens");
  if (tokens == 0) return QFG_OK;
  QFG_CHECK(CheckHeads(name, "k", k, ldk, c.cache.heads, c.cache.dim, elem));
  QFG_CHECK(CheckHeads(name, "v", v, ldv, c.cache.heads, c.cache.dim, elem));
  if (slots == nullptr || !On(slots, 8)) return Refuse(name, "no slots");
  c.dtype = dtype;
  c.dim = c.cache.dim;
  c.k = k;
  c.ldk = ldk;
  c.kv_heads = c.cache.heads;
  c.v = v;
  c.ldv = ldv;
  c.tokens = tokens;
  c.slots = slots;
  return Launched(name, qfg::LaunchHeadRows(c, static_cast<cudaStream_t>(stream)));
}

namespace {

int CheckTable(const char* name, const int32_t* table, int64_t ld_table, int64_t seqs, int64_t most_pages, const qfg::KvCacheView& cache) {
  if (seqs < 0 || seqs > 65536) return Refuse(name, "at most 65536 sequences");
  if (most_pages < 0 || most_pages > INT_MAX / cache.page) return Refuse(name, "a sequence may have at most 2147483647 tokens");
  if (ld_table < most_pages) return Refuse(name, "the rows of the table overlap");
  if (seqs > 0 && ((most_pages > 0 && table == nullptr) || !On(table, 4))) return Refuse(name, "no table");
  return QFG_OK;
}

}  // namespace

int qfg_cache_read(const qfg_kv_cache* cache, const int32_t* table, int64_t ld_table, int64_t seqs, int64_t most_pages, const int32_t* offsets, int64_t rows,
                   int dtype, void* k_out, void* v_out, void* stream) {
  const char* const name = "CacheRead";
  qfg::CacheReadCall c;
  QFG_CHECK(CheckCache(name, cache, &c.cache));
  if (BytesOf(dtype) == 0) return Refuse(name, "the rows must be BF16/FP16/FP32");
  QFG_CHECK(CheckTable(name, table, ld_table, seqs, most_pages, c.cache));
  if (rows < 0 || rows > INT_MAX) return Refuse(name, "bad number of rows");
  if (rows == 0 || seqs == 0) return QFG_OK;
  if (offsets == nullptr || !On(offsets, 4)) return Refuse(name, "no offsets");
  if (k_out == nullptr || v_out == nullptr || !On(k_out, 16) || !On(v_out, 16)) return Refuse(name, "the outputs must begin on 16 bytes");
  c.table = table;
  c.ld_table = ld_table;
  c.seqs = static_cast<int>(seqs);
  c.most_pages = static_cast<int>(most_pages);
  c.offsets = offsets;
  c.rows = rows;
  c.dtype = dtype;
  c.k_out = k_out;
  c.v_out = v_out;
  return Launched(name, qfg::LaunchCacheRead(c, static_cast<cudaStream_t>(stream)));
}

namespace {

int AttentionCall(const qfg_kv_cache* cache, int64_t seqs, int64_t tokens, int64_t q_heads, int64_t most_pages, qfg::CacheAttentionCall* c) {
  const char* const name = "CacheAttention";
  QFG_CHECK(CheckCache(name, cache, &c->cache));
  if (seqs < 0 || seqs > 65536) return Refuse(name, "at most 65536 sequences");
  if (tokens < 0 || tokens > 1024) return Refuse(name, "at most 1024 tokens of a sequence attend in one call");
  if (q_heads < 1 || q_heads > kMostHeads || q_heads % c->cache.heads != 0) return Refuse(name, "the query heads must be a multiple of the cache's, up to 4096");
  if (most_pages < 0 || most_pages > INT_MAX / c->cache.page) return Refuse(name, "a sequence may have at most 2147483647 tokens");
  // what shares of it are counted in
  const int64_t room = seqs * most_pages * c->cache.page, rows = tokens * (q_heads / c->cache.heads);
  if (room > int64_t{1} << 34 || room > (int64_t{1} << 42) / (c->cache.heads * (rows / 8 + 1))) return Refuse(name, "the table is too large");
  c->seqs = static_cast<int>(seqs);
  c->tokens = static_cast<int>(tokens);
  c->q_heads = static_cast<int>(q_heads);
  c->most_pages = static_cast<int>(most_pages);
  return QFG_OK;
}

}  // namespace

int qfg_cache_attention_workspace_bytes(const qfg_kv_cache* cache, int64_t seqs, int64_t tokens, int64_t q_heads, int64_t most_pages, size_t* bytes) {
  if (bytes == nullptr) return Refuse("CacheAttention", "null argument");
  qfg::CacheAttentionCall c;
  *bytes = 0;
  QFG_CHECK(AttentionCall(cache, seqs, tokens, q_heads, most_pages, &c));
  if (seqs > 0 && tokens > 0) *bytes = qfg::CacheAttentionWorkspace(c);
  return QFG_OK;
}

int qfg_cache_attention(int dtype, const void* q, int64_t ld_seq, int64_t ld_token, int64_t seqs, int64_t tokens, int64_t q_heads, const qfg_kv_cache* cache,
                        const int32_t* table, int64_t ld_table, int64_t most_pages, const int32_t* lengths, float scale, void* workspace, void* out, float* lse,
                        void* stream) {
  const char* const name = "CacheAttention";
  qfg::CacheAttentionCall c;
  QFG_CHECK(AttentionCall(cache, seqs, tokens, q_heads, most_pages, &c));
  if (dtype != QFG_BFLOAT16 && dtype != QFG_FLOAT16) return Refuse(name, "q must be BF16/FP16");
  QFG_CHECK(CheckTable(name, table, ld_table, seqs, most_pages, c.cache));
  if (!Scale(scale)) return Refuse(name, "the scale must be positive and finite");
  if (seqs == 0 || tokens == 0) return QFG_OK;
  if (q == nullptr || out == nullptr || lengths == nullptr || !On(lengths, 4) || !On(lse, 4)) return Refuse(name, "null or misaligned argument");
  if (!On(q, 16) || !On(out, 16) || ld_seq % 8 != 0 || ld_token % 8 != 0) return Refuse(name, "q and the output must lie on 16 bytes, token by token");
  if ((tokens > 1 && ld_token < q_heads * c.cache.dim) || (seqs > 1 && ld_seq < q_heads * c.cache.dim)) return Refuse(name, "the rows of q overlap");
  const size_t need = qfg::CacheAttentionWorkspace(c);
  if (need > 0 && (workspace == nullptr || !On(workspace, 16))) return Refuse(name, "the workspace must begin on 16 bytes");
  c.dtype = dtype;
  c.q = q;
  c.ld_seq = ld_seq;
  c.ld_token = ld_token;
  c.table = table;
  c.ld_table = ld_table;
  c.lengths = lengths;
  c.scale = scale;
  c.workspace = workspace;
  c.out = out;
  c.lse = lse;
  return Launched(name, qfg::LaunchCacheAttention(c, static_cast<cudaStream_t>(stream)));
}

int qfg_prompt_attention(int dtype, const void* q, int64_t ldq, int64_t q_rows, int64_t q_heads, const void* k, int64_t ldk, const void* v, int64_t ldv,
                         int64_t k_rows, int64_t kv_heads, int64_t head_dim, const int32_t* q_offsets, const int32_t* k_offsets, int64_t seqs, int causal,
                         float scale, void* out, float* lse, void* stream) {
  const char* const name = "PromptAttention";
  if (dtype != QFG_BFLOAT16 && dtype != QFG_FLOAT16) return Refuse(name, "heads must be BF16/FP16");
  if (head_dim != 64 && head_dim != 128) return Refuse(name, "heads must have 64 or 128 channels");
  if (seqs < 0 || seqs > 65536) return Refuse(name, "at most 65536 sequences");
  if (q_rows < 0 || k_rows < 0 || q_rows > INT_MAX / 2 || k_rows > INT_MAX / 2) return Refuse(name, "bad number of rows");
  if (q_heads < 1 || kv_heads < 1 || q_heads > kMostHeads || q_heads % kv_heads != 0) return Refuse(name, "the query heads must be a multiple of the key heads, up to 4096");
  if (!Scale(scale)) return Refuse(name, "the scale must be positive and finite");
  if (q_rows == 0 || seqs == 0) return QFG_OK;
  QFG_CHECK(CheckHeads(name, "q", q, ldq, q_heads, head_dim, 16));
  if (k_rows > 0) {
    QFG_CHECK(CheckHeads(name, "k", k, ldk, kv_heads, head_dim, 16));
    QFG_CHECK(CheckHeads(name, "v", v, ldv, kv_heads, head_dim, 16));
  }
  if (ldq % 8 != 0 || (k_rows > 0 && (ldk % 8 != 0 || ldv % 8 != 0))) return Refuse(name, "tokens must lie on 16 bytes");
  if (q_offsets == nullptr || k_offsets == nullptr || !On(q_offsets, 4) || !On(k_offsets, 4)) return Refuse(name, "no offsets");
  if (out == nullptr || !On(out, 16) || !On(lse, 4)) return Refuse(name, "the output must begin on 16 bytes");
  qfg::PromptCall c;
  c.dtype = dtype;
  c.dim = static_cast<int>(head_dim);
  c.q_heads = static_cast<int>(q_heads);
  c.kv_heads = static_cast<int>(kv_heads);
  c.seqs = static_cast<int>(seqs);
  c.q = q;
  c.k = k;
  c.v = v;
  c.ldq = ldq;
  c.ldk = ldk;
  c.ldv = ldv;
  c.q_rows = q_rows;
  c.k_rows = k_rows;
  c.q_offsets = q_offsets;
  c.k_offsets = k_offsets;
  c.causal = causal != 0;
  c.scale = scale;
  c.out = out;
  c.lse = lse;
  c.give_up = g_prompt_give_up.load(std::memory_order_relaxed);
  return Launched(name, qfg::LaunchPromptAttention(c, static_cast<cudaStream_t>(stream)));
}

int qfg_prompt_attention_set_option(const char* key, const char* value) {
  if (key == nullptr || value == nullptr) return Refuse("PromptAttention", "null argument");
  if (std::strcmp(key, "give_up") != 0) return Refuse("PromptAttention", std::string("unknown option ") + key);
  g_prompt_give_up.store(std::atoi(value) != 0, std::memory_order_relaxed);
  return QFG_OK;
}
