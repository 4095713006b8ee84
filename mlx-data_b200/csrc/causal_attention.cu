// Attention over a cache and attention in a window: entry points, checks, launches.
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstring>

#include "causal.h"

namespace mlxd {

namespace {

// Tensors as the copies into shared memory want them: 16-byte units throughout.  Strides of dimensions that are not
// stepped along do not matter.
bool aligned(const Heads& h, int64_t batch, int64_t tokens, int64_t heads) {
  return reinterpret_cast<uintptr_t>(h.data) % 16 == 0 && (batch <= 1 || h.batch % 8 == 0) && (tokens <= 1 || h.token % 8 == 0) &&
         (heads <= 1 || h.head % 8 == 0);
}

Heads heads_of(const mlxd_heads& h) {
  return Heads{static_cast<char*>(h.data), h.stride_batch, h.stride_token, h.stride_head};
}

// What both descriptors have.
template <class Desc>
int sizes_of(const char* entry, const Desc* d, CausalParams& p) {
  const auto bad = [&](const std::string& what) { return fail(MLXD_ERR_INVALID, std::string(entry) + ": " + what); };
  if (!d) return bad("no descriptor");
  if (d->dtype != MLXD_BF16 && d->dtype != MLXD_F16) return bad("tensors must be bfloat16 or float16");
  if (d->batch < 0 || d->tokens < 0) return bad("negative size");
  if (d->q_heads < 1 || d->kv_heads < 1 || d->q_heads % d->kv_heads) {
    return bad("q_heads must be a multiple of kv_heads (got " + std::to_string(d->q_heads) + " and " + std::to_string(d->kv_heads) + ")");
  }
  if (d->head_dim < 8 || d->head_dim % 8 || d->head_dim > MLXD_CROSS_MAX_HEAD_DIM) {
    return bad("head_dim must be a multiple of 8 up to " + std::to_string(MLXD_CROSS_MAX_HEAD_DIM) + " (got " + std::to_string(d->head_dim) + ")");
  }
  if (d->tokens >= kMaxPlaces) return bad("2^30 tokens or more");
  if (static_cast<int64_t>(d->batch) * d->q_heads > (1 << 24) || static_cast<int64_t>(d->batch) * d->q_heads * d->tokens > (int64_t{1} << 33)) {
    return bad("too many rows");
  }
  if (d->window < 0 || d->sinks < 0) return bad("window and sinks must not be negative");
  std::memset(&p, 0, sizeof(p));
  p.batch = d->batch;
  p.tokens = d->tokens;
  p.q_heads = d->q_heads;
  p.kv_heads = d->kv_heads;
  p.group = d->q_heads / d->kv_heads;
  p.head_dim = d->head_dim;
  p.scale = d->scale;
  p.window = d->window ? d->window : INT_MAX;
  p.sinks = d->window ? d->sinks : 0;
  return MLXD_OK;
}

// What both calls check beyond sizes.
template <class Desc>
int common_of(const char* entry, const Desc* d, CausalParams& p) {
  const auto bad = [&](const std::string& what) { return fail(MLXD_ERR_INVALID, std::string(entry) + ": " + what); };
  if (!std::isfinite(d->scale) || d->scale <= 0) return bad("scale must be positive and finite");
  // a kernel reads and writes whole elements, and a misaligned one is a fault
  if (!on_boundary(d->lse, 4)) return bad("lse does not start on a multiple of 4 bytes");
  if (!on_boundary(d->workspace, 16)) return bad("workspace must start on 16 bytes");
  p.q = heads_of(d->q);
  p.out = heads_of(d->out);
  p.lse = d->lse;
  return MLXD_OK;
}

int tensor_of(const char* entry, const char* name, const Heads& h, int64_t batch, int64_t tokens, int64_t heads) {
  const auto bad = [&](const std::string& what) { return fail(MLXD_ERR_INVALID, std::string(entry) + ": " + name + what); };
  if (!batch || !tokens) return MLXD_OK;   // an empty tensor
  if (!h.data) return bad(" is needed");
  if (!aligned(h, batch, tokens, heads)) return bad(" must start on 16 bytes and have strides that are multiples of 8");
  return MLXD_OK;
}

// Maps of queries and results: boxes of 64 elements of a tile's rows.
int rows_map(const char* entry, const CausalParams& p, const RowTiles& r, const Heads& h, int dtype, CUtensorMap* map) {
  const uint64_t sizes[5] = {static_cast<uint64_t>(p.head_dim), static_cast<uint64_t>(p.group), static_cast<uint64_t>(p.tokens),
                             static_cast<uint64_t>(p.kv_heads), static_cast<uint64_t>(p.batch)};
  const int64_t strides[5] = {1, h.head, h.token, h.head * p.group, h.batch};
  const uint32_t box[5] = {64, static_cast<uint32_t>(r.heads), static_cast<uint32_t>(r.tokens), 1, 1};
  return tile_map(entry, dtype, p.device, h.data, 5, sizes, strides, box, map);
}

// Of keys and values: boxes of 64 elements of 128 tokens, or of as many as a page has.
int keys_map(const char* entry, const CausalParams& p, const Heads& h, int64_t major, int64_t minor, int dtype, CUtensorMap* map) {
  const uint64_t sizes[4] = {static_cast<uint64_t>(p.head_dim), static_cast<uint64_t>(minor), static_cast<uint64_t>(p.kv_heads), static_cast<uint64_t>(major)};
  const int64_t strides[4] = {1, h.token, h.head, h.batch};
  const uint32_t box[4] = {64, p.cache.page_size ? static_cast<uint32_t>(std::min(p.cache.page_size, 128)) : 128u, 1, 1};
  return tile_map(entry, dtype, p.device, h.data, 4, sizes, strides, box, map);
}

int forward(const char* entry, CausalParams& p, int dtype, bool paged, void* workspace, size_t workspace_bytes, int device, void* stream) {
  p.device = device;
  int sms = 0;
  int rc = device_sms(device, &sms);
  if (rc != MLXD_OK) return rc;
  ForwardParams f = forward_plan(p, paged, sms);
  const size_t need = forward_workspace(f);
  if (need && (!workspace || workspace_bytes < need)) return fail(MLXD_ERR_INVALID, std::string(entry) + ": workspace too small");
  MLXD_ON_DEVICE(device);
  rc = status_word(device, &f.p.status);
  const int64_t rows = static_cast<int64_t>(p.batch) * p.q_heads * p.tokens;
  f.part_out = static_cast<float*>(workspace);
  f.part_lse = f.part_out + (need ? f.parts * rows * p.head_dim : 0);
  const auto join = [&] {
    if (f.parts > 1) MLXD_CUDA(launch_causal_join(f, dtype, static_cast<cudaStream_t>(stream)));
    return static_cast<int>(MLXD_OK);
  };
  if (rc != MLXD_OK) return rc;
  if (f.steps) {
    MLXD_CUDA(launch_causal_step(f, dtype, static_cast<cudaStream_t>(stream)));
    return join();
  }
  CausalMaps maps;
  const int64_t major = paged ? p.cache.pages : p.batch, minor = paged ? p.cache.page_size : p.tokens;
  rc = rows_map(entry, p, f.rows, p.q, dtype, &maps.q);
  if (rc == MLXD_OK && major) rc = keys_map(entry, p, p.k, major, minor, dtype, &maps.k);   // without pages there is nothing to read
  if (rc == MLXD_OK && major) rc = keys_map(entry, p, p.v, major, minor, dtype, &maps.v);
  if (rc != MLXD_OK) return rc;
  MLXD_CUDA(launch_causal_forward(f, maps, paged, dtype, static_cast<cudaStream_t>(stream)));
  return join();
}

int cached_params(const char* entry, const mlxd_cached_desc* d, CausalParams& p) {
  const auto bad = [&](const std::string& what) { return fail(MLXD_ERR_INVALID, std::string(entry) + ": " + what); };
  int rc = sizes_of(entry, d, p);
  if (rc == MLXD_OK) rc = common_of(entry, d, p);
  if (rc == MLXD_OK) rc = cache_of(entry, d->cache, d->batch, &p.cache);
  if (rc != MLXD_OK) return rc;
  p.k = pages_of(d->cache.k);
  p.v = pages_of(d->cache.v);
  rc = tensor_of(entry, "q", p.q, p.batch, p.tokens, p.q_heads);
  if (rc == MLXD_OK) rc = tensor_of(entry, "out", p.out, p.batch, p.tokens, p.q_heads);
  if (rc == MLXD_OK) rc = tensor_of(entry, "k_pages", p.k, d->cache.pages, d->cache.page_size, p.kv_heads);
  if (rc == MLXD_OK) rc = tensor_of(entry, "v_pages", p.v, d->cache.pages, d->cache.page_size, p.kv_heads);
  if (rc != MLXD_OK) return rc;
  if (d->tree && p.tokens > (1 << 16)) return bad("a tree of more than 65536 tokens");
  p.tree = d->tree;
  p.tree_batch = d->tree_stride_batch;
  p.tree_token = d->tree_stride_token;
  return MLXD_OK;
}

int window_params(const char* entry, const mlxd_window_desc* d, bool backward, CausalParams& p) {
  const auto bad = [&](const std::string& what) { return fail(MLXD_ERR_INVALID, std::string(entry) + ": " + what); };
  int rc = sizes_of(entry, d, p);
  if (rc == MLXD_OK) rc = common_of(entry, d, p);
  if (rc != MLXD_OK) return rc;
  if (d->lengths && d->lengths_dtype != MLXD_I32 && d->lengths_dtype != MLXD_I64) return bad("lengths must be int32 or int64");
  if (d->lengths && !on_boundary(d->lengths, dtype_bytes(d->lengths_dtype))) return bad("lengths do not start on a multiple of their element's size");
  p.lengths = d->lengths;
  p.lengths_dtype = d->lengths_dtype;
  p.k = heads_of(d->k);
  p.v = heads_of(d->v);
  p.dout = heads_of(d->dout);
  p.dq = heads_of(d->dq);
  p.dk = heads_of(d->dk);
  p.dv = heads_of(d->dv);
  p.lse_grad = d->lse_grad;
  const struct { const Heads* h; bool query; const char* name; } need[] = {
      {&p.q, true, "q"}, {&p.k, false, "k"}, {&p.v, false, "v"}, {&p.out, true, "out"},
      {&p.dout, true, "dout"}, {&p.dq, true, "dq"}, {&p.dk, false, "dk"}, {&p.dv, false, "dv"}};
  for (int i = 0; i < (backward ? 8 : 4); i++) {
    rc = tensor_of(entry, need[i].name, *need[i].h, p.batch, p.tokens, need[i].query ? p.q_heads : p.kv_heads);
    if (rc != MLXD_OK) return rc;
  }
  if (backward) {
    if (p.batch && p.tokens && !d->lse) return bad("lse is needed");
    if (!on_boundary(d->lse_grad, 4)) return bad("lse_grad does not start on a multiple of 4 bytes");
    if (p.batch && p.tokens && (!d->workspace || d->workspace_bytes < backward_workspace(p))) return bad("workspace too small");
  }
  return MLXD_OK;
}

int window_call(const char* entry, int device, void* stream, const mlxd_window_desc* d, bool backward) {
  CausalParams p;
  int rc = window_params(entry, d, backward, p);
  if (rc != MLXD_OK) return rc;
  if (!p.batch || !p.tokens) return MLXD_OK;
  if (!backward) return forward(entry, p, d->dtype, false, d->workspace, d->workspace_bytes, device, stream);
  MLXD_ON_DEVICE(device);
  p.device = device;
  rc = status_word(device, &p.status);
  const RowTiles rows = row_tiles(p);
  CausalMaps maps;
  const struct { const Heads* h; bool query; CUtensorMap* map; } all[] = {
      {&p.q, true, &maps.q}, {&p.dout, true, &maps.dout}, {&p.k, false, &maps.k}, {&p.v, false, &maps.v}};
  for (const auto& x : all) {
    if (rc == MLXD_OK) rc = x.query ? rows_map(entry, p, rows, *x.h, d->dtype, x.map) : keys_map(entry, p, *x.h, p.batch, p.tokens, d->dtype, x.map);
  }
  if (rc != MLXD_OK) return rc;
  MLXD_CUDA(launch_causal_backward(p, d->workspace, maps, d->dtype, static_cast<cudaStream_t>(stream)));
  return MLXD_OK;
}

int forward_bytes(const CausalParams& p, bool paged, int device, size_t* bytes) {
  *bytes = 0;
  if (!p.batch || !p.tokens) return MLXD_OK;
  int sms = 0;
  const int rc = device_sms(device, &sms);
  if (rc == MLXD_OK) *bytes = forward_workspace(forward_plan(p, paged, sms));
  return rc;
}

}  // namespace

int cache_of(const char* entry, const mlxd_cache& c, int batch, CacheParams* p) {
  const auto bad = [&](const std::string& what) { return fail(MLXD_ERR_INVALID, std::string(entry) + ": " + what); };
  if (c.pages < 0 || c.table_width < 0) return bad("negative size");
  if (c.page_size < 8 || (c.page_size & (c.page_size - 1))) return bad("page_size must be a power of two from 8 on (got " + std::to_string(c.page_size) + ")");
  if (static_cast<int64_t>(c.table_width) * c.page_size > kMaxPlaces) return bad("more than 2^30 places in a row of page_table");
  const auto integers = [&](const char* name, const void* x, int dtype) {
    if (dtype != MLXD_I32 && dtype != MLXD_I64) return bad(std::string(name) + " must be int32 or int64");
    if (!on_boundary(x, dtype_bytes(dtype))) return bad(std::string(name) + " does not start on a multiple of its element's size");
    return static_cast<int>(MLXD_OK);
  };
  int rc = integers("page_table", c.page_table, c.page_table_dtype);
  if (rc == MLXD_OK) rc = integers("lengths", c.lengths, c.lengths_dtype);
  if (rc == MLXD_OK && c.counts) rc = integers("counts", c.counts, c.counts_dtype);
  if (rc != MLXD_OK) return rc;
  if (batch && !c.lengths) return bad("lengths are needed");
  if (batch && c.table_width && !c.page_table) return bad("page_table is needed");
  p->table = c.page_table;
  p->lengths = c.lengths;
  p->counts = c.counts;
  p->table_stride = c.page_table_stride;
  p->table_width = c.pages ? c.table_width : 0;   // a pool of no pages has no places
  p->pages = c.pages;
  p->page_size = c.page_size;
  p->page_shift = __builtin_ctz(static_cast<unsigned>(c.page_size));
  p->capacity = p->table_width * c.page_size;
  p->table_dtype = c.page_table_dtype;
  p->lengths_dtype = c.lengths_dtype;
  p->counts_dtype = c.counts_dtype;
  return MLXD_OK;
}

}  // namespace mlxd

using namespace mlxd;

extern "C" int mlxd_cached_attention_workspace(int device, const mlxd_cached_desc* d, size_t* bytes) {
  return guarded("cached_attention_workspace", [&] {
    CausalParams p;
    int rc = sizes_of("cached_attention_workspace", d, p);
    if (rc != MLXD_OK) return rc;
    if (!bytes) return fail(MLXD_ERR_INVALID, "cached_attention_workspace: no place for the result");
    rc = cache_of("cached_attention_workspace", d->cache, d->batch, &p.cache);
    if (rc != MLXD_OK) return rc;
    return forward_bytes(p, true, device, bytes);
  });
}

extern "C" int mlxd_cached_attention(int device, void* cuda_stream, const mlxd_cached_desc* d) {
  return guarded("cached_attention", [&] {
    CausalParams p;
    const int rc = cached_params("cached_attention", d, p);
    if (rc != MLXD_OK) return rc;
    if (!p.batch || !p.tokens) return static_cast<int>(MLXD_OK);
    return forward("cached_attention", p, d->dtype, true, d->workspace, d->workspace_bytes, device, cuda_stream);
  });
}

extern "C" int mlxd_window_attention_workspace(int device, const mlxd_window_desc* d, int backward, size_t* bytes) {
  return guarded("window_attention_workspace", [&] {
    CausalParams p;
    const int rc = sizes_of("window_attention_workspace", d, p);
    if (rc != MLXD_OK) return rc;
    if (!bytes) return fail(MLXD_ERR_INVALID, "window_attention_workspace: no place for the result");
    if (!backward) return forward_bytes(p, false, device, bytes);
    *bytes = p.batch && p.tokens ? backward_workspace(p) : 0;
    return static_cast<int>(MLXD_OK);
  });
}

extern "C" int mlxd_window_attention(int device, void* cuda_stream, const mlxd_window_desc* d) {
  return guarded("window_attention", [&] { return window_call("window_attention", device, cuda_stream, d, false); });
}

extern "C" int mlxd_window_attention_backward(int device, void* cuda_stream, const mlxd_window_desc* d) {
  return guarded("window_attention_backward", [&] { return window_call("window_attention_backward", device, cuda_stream, d, true); });
}
