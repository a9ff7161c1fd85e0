// The paged key-value cache above the C ABI: checks, allocation and launch.  These operators have no gradients.
#include "functions.h"

namespace tfb_host {

static void check_plain(const char* what, std::initializer_list<const Tensor*> inputs) {
  if (needs_node(inputs)) throw ArgumentError(std::string(what) + ": no gradients: call it under torch.no_grad()");
  const Tensor* first = nullptr;
  for (const Tensor* t : inputs) {
    if (!t->defined()) continue;
    if (!t->is_cuda()) throw ArgumentError(std::string(what) + ": expected CUDA tensors");
    if (!first) first = t;
    if (t->device() != first->device()) throw ArgumentError(std::string(what) + ": tensors on different devices");
  }
}

// Strides of a dimension of one entry say nothing and may be anything.
static int64_t step(const Tensor& t, int64_t dim) { return t.size(dim) > 1 ? t.stride(dim) : 0; }
static Tensor unit_inner(const Tensor& t) { return t.size(-1) > 1 && t.stride(-1) != 1 ? t.contiguous() : t; }
static const int* ints(const Tensor& t) { return t.defined() ? static_cast<const int*>(t.data_ptr()) : nullptr; }
static float* floats(const Tensor& t) { return t.defined() ? static_cast<float*>(t.data_ptr()) : nullptr; }

struct Pool {
  int64_t pages, heads, page, hd, strides[3];
};
static Pool pool_of(const Tensor& k, const Tensor& v, const Tensor& mass, const Tensor& positions) {
  TFB_ASSERT(k.defined() && v.defined() && k.dim() == 4 && k.sizes() == v.sizes(),
             "key and value pages are (pages, heads, page, head_dim) tensors of one shape");
  TFB_ASSERT((k.scalar_type() == at::kHalf || k.scalar_type() == at::kBFloat16) && v.scalar_type() == k.scalar_type(),
             "the pages hold matching fp16/bf16");
  TFB_ASSERT(k.size(3) == 32 || k.size(3) == 64 || k.size(3) == 128, "Only head_dims of [32,64,128] are supported.");
  TFB_ASSERT(k.size(0) > 0 && k.size(1) > 0 && k.size(2) > 0, "the cache has no pages");
  TFB_ASSERT(k.stride(3) == 1 && v.stride(3) == 1, "the pages need a unit stride on head_dim");
  Pool p{k.size(0), k.size(1), k.size(2), k.size(3), {step(k, 0), step(k, 1), step(k, 2)}};
  for (int i = 0; i < 3; ++i) {
    TFB_ASSERT(step(v, i) == p.strides[i], "key and value pages need the same strides");
    TFB_ASSERT(k.size(i) == 1 || p.strides[i] > 0, "the pages overlap");
  }
  for (const Tensor* t : {&mass, &positions})
    if (t->defined())
      TFB_ASSERT(t->dim() == 3 && t->size(0) == p.pages && t->size(1) == p.heads && t->size(2) == p.page && t->is_contiguous(),
                 "mass and positions are contiguous (pages, heads, page) tensors");
  TFB_ASSERT(!mass.defined() || mass.scalar_type() == at::kFloat, "masses are fp32");
  TFB_ASSERT(!positions.defined() || positions.scalar_type() == at::kInt, "positions are int32");
  return p;
}

struct Table {
  const int* p;
  int64_t width, ld;
};
static Table table_of(const Tensor& t, int64_t batch) {
  TFB_ASSERT(t.defined() && t.dim() == 2 && t.size(0) == batch && t.size(1) > 0 && t.scalar_type() == at::kInt,
             "the tables are a (batch, pages) int32 tensor");
  TFB_ASSERT(t.size(1) == 1 || t.stride(1) == 1, "the tables need a unit stride along a row");
  TFB_ASSERT(batch <= 1 || t.stride(0) >= t.size(1), "the tables' rows overlap");
  return {static_cast<const int*>(t.data_ptr()), t.size(1), batch > 1 ? t.stride(0) : t.size(1)};
}
static void check_per_sequence(const Tensor& t, int64_t batch, const char* what) {
  if (t.defined() && !(t.dim() == 1 && t.size(0) == batch && t.scalar_type() == at::kInt && t.is_contiguous()))
    throw ArgumentError(std::string(what) + ": expected a contiguous (batch,) int32 tensor");
}

Tensor paged_attention(const Tensor& q_, const Tensor& k_pages, const Tensor& v_pages, const Tensor& tables, const Tensor& lengths,
                       const Tensor& key_, const Tensor& value_, const Tensor& slopes, int64_t rounded,
                       const Tensor& query_positions, const Tensor& mass, const Tensor& positions, const Tensor& mass_out_) {
  check_plain("paged_attention", {&q_, &k_pages, &v_pages, &tables, &lengths, &key_, &value_, &slopes, &query_positions, &mass,
                                  &positions, &mass_out_});
  BodyGuard guard;
  const Pool pool = pool_of(k_pages, v_pages, mass, positions);
  TFB_ASSERT(q_.defined() && q_.dim() == 3 && q_.size(2) == pool.hd, "the query is a (batch, heads, head_dim) tensor");
  TFB_ASSERT(q_.scalar_type() == k_pages.scalar_type(), "the query has the pages' type");
  const int64_t B = q_.size(0), heads = q_.size(1);
  TFB_ASSERT(heads > 0 && heads % pool.heads == 0, "the query heads are a multiple of the cache's heads");
  const Table table = table_of(tables, B);
  TFB_ASSERT(lengths.defined(), "lengths: expected a contiguous (batch,) int32 tensor");
  check_per_sequence(lengths, B, "lengths");
  check_per_sequence(query_positions, B, "query_positions");
  TFB_ASSERT(key_.defined() == value_.defined(), "a new key comes with a value");
  Tensor key, value;
  if (key_.defined()) {
    TFB_ASSERT(key_.dim() == 3 && key_.size(0) == B && key_.size(1) == pool.heads && key_.size(2) == pool.hd &&
                   value_.sizes() == key_.sizes(),
               "new keys and values are (batch, cache heads, head_dim) tensors");
    TFB_ASSERT(key_.scalar_type() == k_pages.scalar_type() && value_.scalar_type() == k_pages.scalar_type(),
               "new keys and values have the pages' type");
    key = unit_inner(key_);
    value = unit_inner(value_);
  }
  TFB_ASSERT(!slopes.defined() || (slopes.dim() == 1 && slopes.size(0) == heads && slopes.scalar_type() == at::kFloat &&
                                   slopes.is_contiguous()),
             "the slopes are a contiguous (heads,) fp32 tensor");
  const Tensor mass_out = mass_out_.defined() ? mass_out_ : mass;
  TFB_ASSERT(mass.defined() || !mass_out.defined(), "mass_out without mass");
  if (mass_out_.defined())
    TFB_ASSERT(mass_out_.sizes() == mass.sizes() && mass_out_.scalar_type() == at::kFloat && mass_out_.is_contiguous(),
               "mass_out is like mass");
  const Tensor q = unit_inner(q_);
  Tensor out = at::empty({B, heads, pool.hd}, q.options());
  if (B == 0) return out;
  const int64_t group = heads / pool.heads;
  const int64_t bytes = mass.defined() ? tfb_paged_attention_scratch_bytes(B, pool.heads, group, table.width * pool.page) : 0;
  Tensor scratch;
  if (bytes) scratch = at::empty({bytes}, q.options().dtype(at::kByte));
  const cudaStream_t stream = current_stream(q);
  const Tensor ws = gemm_workspace(q.device(), stream);
  const int64_t sq[2] = {step(q, 0), step(q, 1)}, so[2] = {heads * pool.hd, pool.hd};
  int64_t sk[2] = {0, 0}, sv[2] = {0, 0};
  if (key.defined())
    for (int i = 0; i < 2; ++i) {
      sk[i] = step(key, i);
      sv[i] = step(value, i);
    }
  check(tfb_paged_attention(q.data_ptr(), key.defined() ? key.data_ptr() : nullptr, value.defined() ? value.data_ptr() : nullptr,
                            out.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), table.p, ints(lengths), ints(query_positions),
                            const_cast<int*>(ints(positions)), floats(mass), floats(mass_out), floats(slopes), (int)rounded, B,
                            pool.heads, group, pool.hd, pool.pages, pool.page, table.width, table.ld, pool.strides, sq, sk, sv, so,
                            ws.data_ptr(), ws.numel(), bytes ? scratch.data_ptr() : nullptr, bytes, dtype_code(q.scalar_type()),
                            stream));
  return out;
}

void cache_append(const Tensor& k_pages, const Tensor& v_pages, const Tensor& tables, const Tensor& lengths, const Tensor& key_,
                  const Tensor& value_, const Tensor& counts, const Tensor& mass, const Tensor& positions, const Tensor& key_mass_,
                  const Tensor& first_positions) {
  check_plain("cache_append", {&k_pages, &v_pages, &tables, &lengths, &key_, &value_, &counts, &mass, &positions, &key_mass_,
                               &first_positions});
  BodyGuard guard;
  const Pool pool = pool_of(k_pages, v_pages, mass, positions);
  TFB_ASSERT(key_.defined() && value_.defined() && key_.dim() == 4 && key_.sizes() == value_.sizes() &&
                 key_.size(1) == pool.heads && key_.size(3) == pool.hd,
             "keys and values are (batch, cache heads, T, head_dim) tensors");
  TFB_ASSERT(key_.scalar_type() == k_pages.scalar_type() && value_.scalar_type() == k_pages.scalar_type(),
             "keys and values have the pages' type");
  const int64_t B = key_.size(0), T = key_.size(2);
  const Table table = table_of(tables, B);
  TFB_ASSERT(lengths.defined(), "lengths: expected a contiguous (batch,) int32 tensor");
  check_per_sequence(lengths, B, "lengths");
  check_per_sequence(counts, B, "counts");
  check_per_sequence(first_positions, B, "first_positions");
  Tensor key_mass;
  if (key_mass_.defined()) {
    TFB_ASSERT(mass.defined(), "masses of the keys, and the cache has none");
    TFB_ASSERT(key_mass_.dim() == 3 && key_mass_.size(0) == B && key_mass_.size(1) == pool.heads && key_mass_.size(2) == T &&
                   key_mass_.scalar_type() == at::kFloat,
               "the keys' masses are a (batch, cache heads, T) fp32 tensor");
    key_mass = unit_inner(key_mass_);
  }
  if (B == 0 || T == 0) return;
  const Tensor key = unit_inner(key_), value = unit_inner(value_);
  const int64_t sk[3] = {step(key, 0), step(key, 1), step(key, 2)}, sv[3] = {step(value, 0), step(value, 1), step(value, 2)};
  int64_t sm[2] = {0, 0};
  if (key_mass.defined())
    for (int i = 0; i < 2; ++i) sm[i] = step(key_mass, i);
  check(tfb_cache_append(key.data_ptr(), value.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), table.p, ints(lengths),
                         ints(counts), ints(first_positions), floats(mass), const_cast<int*>(ints(positions)), floats(key_mass), B,
                         pool.heads, T, pool.hd, pool.pages, pool.page, table.width, table.ld, pool.strides, sk, sv, sm,
                         dtype_code(key.scalar_type()), current_stream(key)));
}

// What a tensor map can describe: 16-byte aligned rows, no repetition; strides of dimensions of one entry made to fit.
static bool mapped(const Tensor& t, int64_t (&s)[3]) {
  bool ok = t.stride(3) == 1 && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
  for (int i = 0; i < 3; ++i) {
    s[i] = t.size(i) > 1 ? t.stride(i) : t.size(3);
    ok = ok && s[i] > 0 && s[i] % 8 == 0;
  }
  return ok;
}

Tensor prompt_mass(const Tensor& q_, const Tensor& k_, const Tensor& lse_, const Tensor& counts, const Tensor& slopes, int64_t rounded) {
  check_plain("prompt_mass", {&q_, &k_, &lse_, &counts, &slopes});
  BodyGuard guard;
  TFB_ASSERT(q_.defined() && k_.defined() && q_.dim() == 4 && k_.dim() == 4 && q_.size(0) == k_.size(0) && q_.size(2) == k_.size(2) &&
                 q_.size(3) == k_.size(3) && k_.size(1) > 0 && q_.size(1) > 0 && q_.size(1) % k_.size(1) == 0,
             "q and k are (batch, heads, T, head_dim) tensors, the query heads a multiple of the key heads");
  TFB_ASSERT((q_.scalar_type() == at::kHalf || q_.scalar_type() == at::kBFloat16) && k_.scalar_type() == q_.scalar_type(),
             "prompt_mass expects matching fp16/bf16 inputs");
  const int64_t B = q_.size(0), heads = q_.size(1), T = q_.size(2), hd = q_.size(3), kv_heads = k_.size(1);
  TFB_ASSERT(hd == 32 || hd == 64 || hd == 128, "Only head_dims of [32,64,128] are supported.");
  TFB_ASSERT(lse_.defined() && lse_.dim() == 3 && lse_.size(0) == B && lse_.size(1) == heads && lse_.size(2) == T &&
                 lse_.scalar_type() == at::kFloat,
             "the log-sum-exp is a (batch, heads, T) fp32 tensor");
  check_per_sequence(counts, B, "counts");
  TFB_ASSERT(!slopes.defined() || (slopes.dim() == 1 && slopes.size(0) == heads && slopes.scalar_type() == at::kFloat &&
                                   slopes.is_contiguous()),
             "the slopes are a contiguous (heads,) fp32 tensor");
  Tensor out = at::empty({B, kv_heads, T}, lse_.options());
  if (B == 0 || T == 0) return out;
  Tensor q = q_, k = k_, lse = unit_inner(lse_);
  int64_t sq[3], sk[3];
  if (!mapped(q, sq)) mapped(q = q.clone(at::MemoryFormat::Contiguous), sq);
  if (!mapped(k, sk)) mapped(k = k.clone(at::MemoryFormat::Contiguous), sk);
  const int64_t sl[2] = {step(lse, 0), step(lse, 1)};
  const cudaStream_t stream = current_stream(q);
  const Tensor ws = gemm_workspace(q.device(), stream);
  check(tfb_prompt_mass(q.data_ptr(), k.data_ptr(), floats(lse), ints(counts), floats(slopes), (int)rounded, floats(out), B, kv_heads,
                        heads / kv_heads, T, hd, sq, sk, sl, ws.data_ptr(), ws.numel(), dtype_code(q.scalar_type()), stream));
  return out;
}

Tensor cache_evict(const Tensor& k, const Tensor& v, const Tensor& mass, const Tensor& positions, const Tensor& tables,
                   const Tensor& lengths, const Tensor& next_positions, const Tensor& k_out_, const Tensor& v_out_,
                   const Tensor& mass_out_, const Tensor& positions_out_, const Tensor& out_tables_, int64_t keep, int64_t recent) {
  check_plain("cache_evict", {&k, &v, &mass, &positions, &tables, &lengths, &next_positions, &k_out_, &v_out_, &mass_out_,
                              &positions_out_, &out_tables_});
  BodyGuard guard;
  const Pool pool = pool_of(k, v, mass, positions);
  TFB_ASSERT(mass.defined(), "cache_evict: the cache has no masses");
  TFB_ASSERT(tables.defined() && tables.dim() == 2, "the tables are a (batch, pages) int32 tensor");
  const int64_t B = tables.size(0);
  const Table table = table_of(tables, B);
  TFB_ASSERT(lengths.defined(), "lengths: expected a contiguous (batch,) int32 tensor");
  check_per_sequence(lengths, B, "lengths");
  check_per_sequence(next_positions, B, "next_positions");
  const Tensor& k_out = k_out_.defined() ? k_out_ : k;
  const Tensor& v_out = v_out_.defined() ? v_out_ : v;
  const Tensor& mass_out = mass_out_.defined() ? mass_out_ : mass;
  const Tensor& positions_out = positions_out_.defined() ? positions_out_ : positions;
  const Pool out = pool_of(k_out, v_out, mass_out, positions_out);
  TFB_ASSERT(out.heads == pool.heads && out.hd == pool.hd && k_out.scalar_type() == k.scalar_type(),
             "cache_evict: the outputs have the cache's heads, head_dim and type");
  TFB_ASSERT(positions.defined() == positions_out.defined(), "cache_evict: positions come with positions for the output");
  const Table out_table = out_tables_.defined() ? table_of(out_tables_, B) : table;
  TFB_ASSERT(keep >= 1, "cache_evict: keep: expected at least 1");
  TFB_ASSERT(recent >= 0 && recent <= keep, "cache_evict: recent: expected 0 to keep");
  Tensor left = at::empty({B}, lengths.options());
  if (B == 0) return left;
  const int64_t most = std::min(keep, table.width * pool.page);  // a longer list would never be filled
  const int64_t bytes = tfb_cache_evict_scratch_bytes(B, pool.heads, most);
  Tensor scratch = at::empty({bytes}, lengths.options().dtype(at::kByte));
  check(tfb_cache_evict(k.data_ptr(), v.data_ptr(), floats(mass), ints(positions), table.p, ints(lengths), ints(next_positions),
                        k_out.data_ptr(), v_out.data_ptr(), floats(mass_out), const_cast<int*>(ints(positions_out)), out_table.p,
                        static_cast<int*>(left.data_ptr()), B, pool.heads, pool.hd, most, std::min(recent, most), pool.page,
                        pool.pages, table.width, table.ld, pool.strides, out.page, out.pages, out_table.width, out_table.ld,
                        out.strides, scratch.data_ptr(), bytes, dtype_code(k.scalar_type()), current_stream(k)));
  return left;
}

}  // namespace tfb_host
