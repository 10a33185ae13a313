// dgi/csrc/longctx/bindings.cpp — torch.ops.dgi.* entries of the operators for long caches (dgi/_C_longctx.so): the append that keeps page
// bounds, their rebuilding, page selection, attention over selected pages, attention of drafted trees.
//
// Operands are checked here, on the host, before any launch.  Launches go to the current stream of the operands' device, which is made
// current for them; scratch memory comes from the caching allocator of that stream, a call's own.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime.h>
#include <torch/library.h>

extern "C" {
int dgi_rope_cache_bounds(const void* qkv, long long ld, int T, const int* positions, int max_pos, const float* cos_sin, int nh, int nkv,
                          int hd, int rd, int mode, const int* slots, long long n_slots, void* q_out, void* k_cache, void* v_cache,
                          void* bounds, int block_size, hipStream_t s);
int dgi_page_bounds(const void* k_cache, void* bounds, const int* pages, const int* lens, int n, int num_blocks, int nkv, int hd,
                    int block_size, hipStream_t s);
int dgi_select_pages(const void* q, long long q_stride, const void* bounds, const int* tables, int table_stride, int table_cols, int n_seqs,
                     int num_blocks, const int* ctx, const int* row_seq, int T, int nh, int nkv, int hd, int page, int count, int first,
                     int recent, void* keys, int key_stride, int key_rows, int* out, hipStream_t s);
int dgi_paged_selected(const void* q, long long q_stride, const void* k, const void* v, const int* tables, int table_stride, int table_cols,
                       int n_seqs, int num_blocks, const int* ctx, const int* row_seq, const int* pages, int count, void* out,
                       long long out_stride, float* part_o, float* part_l, int splits, void* plan, int* plan_total, int* plan_rows, int T, int nh,
                       int nkv, int hd, int block_size, float scale, hipStream_t s);
int dgi_tree_rows(const void* q, long long q_stride, const void* k, const void* v, const int* tables, int table_stride, int table_cols,
                   int n_seqs, int num_blocks, int rows, const int* cu, const int* ctx, const void* mask, int mask_stride, int max_nodes,
                   void* out, long long out_stride, float* part_o, float* part_l, int splits, int min_part, int nh, int nkv, int hd,
                   int block_size, float scale, hipStream_t s);
int dgi_tree_tiles(const void* q, long long q_stride, const void* k, const void* v, const int* tables, int table_stride, int table_cols,
                   int n_seqs, int num_blocks, int rows, const int* cu, const int* ctx, const void* mask, int mask_stride, int max_nodes,
                   void* out, long long out_stride, float* part_o, float* part_l, int shares, int least, int nh, int nkv, int hd,
                   int block_size, float scale, hipStream_t s);
}

namespace {

constexpr int64_t kInt = (1ll << 31) - 1;

hipStream_t cur_stream() { return c10::hip::getCurrentHIPStream().stream(); }

void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == 0, "dgi kernel ", what, " failed with code ", rc,
              rc > 0 ? (std::string(" (") + hipGetErrorString((hipError_t)rc) + ")") : std::string());
}

bool aligned(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

// a bf16 operand on `dev` that starts on 16 bytes, and whose gradient nobody waits for
void check_bf16(const at::Tensor& t, const at::Device& dev, const char* op, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.device() == dev, op, ": ", name, " must be on the GPU of the other operands");
  TORCH_CHECK_VALUE(t.scalar_type() == at::kBFloat16, op, ": ", name, " must be bfloat16");
  TORCH_CHECK_VALUE(aligned(t), op, ": ", name, " must start on 16 bytes");
  TORCH_CHECK_VALUE(!(t.requires_grad() && c10::GradMode::is_enabled()), op, ": no gradient goes through ", name);
}

void check_int(const at::Tensor& t, const at::Device& dev, at::ScalarType type, const char* op, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.device() == dev, op, ": ", name, " must be on the GPU of the other operands");
  TORCH_CHECK_VALUE(t.scalar_type() == type && t.is_contiguous(), op, ": ", name, " must be contiguous ", at::toString(type));
}

// rows of heads: [T, >= cols], any row stride that keeps 16 bytes
void check_rows(const at::Tensor& t, int64_t cols, const at::Device& dev, const char* op, const char* name) {
  check_bf16(t, dev, op, name);
  TORCH_CHECK_VALUE(t.dim() == 2 && t.size(1) >= cols && (t.size(0) <= 1 || (t.stride(0) % 8 == 0 && t.stride(0) >= cols)) && t.stride(1) == 1,
                    op, ": ", name, " must be rows of at least ", cols, " values, side by side, that start on 16 bytes");
  TORCH_CHECK_VALUE(t.size(0) <= kInt, op, ": too many rows");
}

void check_heads(int64_t nh, int64_t nkv, int64_t hd, const char* op) {
  TORCH_CHECK_VALUE(nkv > 0 && nh > 0 && nh % nkv == 0 && nh / nkv <= 16, op, ": heads must be 1 to 16 for each kv head");
  TORCH_CHECK_VALUE(hd == 64 || hd == 128 || hd == 256, op, ": heads of 64, 128 or 256 dims");
}

void check_cache(const at::Tensor& c, int64_t nkv, const at::Device& dev, const char* op, const char* name) {
  check_bf16(c, dev, op, name);
  TORCH_CHECK_VALUE(c.dim() == 4 && c.is_contiguous() && c.size(0) > 0 && c.size(0) <= kInt && c.size(1) == nkv && c.size(2) > 0 &&
                        c.size(2) <= (1 << 20),
                    op, ": ", name, " must be contiguous [blocks, kv heads, block size, dims]");
}

void check_bounds(const at::Tensor& b, int64_t nkv, int64_t hd, const at::Device& dev, const char* op) {
  check_bf16(b, dev, op, "bounds");
  TORCH_CHECK_VALUE(b.dim() == 4 && b.is_contiguous() && b.size(0) > 0 && b.size(0) <= kInt && b.size(1) == nkv && b.size(2) == 2 &&
                        b.size(3) == hd,
                    op, ": bounds must be contiguous [blocks, kv heads, 2, dims]");
}

void check_tables(const at::Tensor& t, const at::Device& dev, const char* op) {
  check_int(t, dev, at::kInt, op, "block_tables");
  TORCH_CHECK_VALUE(t.dim() == 2 && t.size(0) <= kInt && t.size(1) <= kInt, op, ": block_tables must be [sequences, pages]");
}

const int* rows_of(const c10::optional<at::Tensor>& row_seq, const at::Tensor& tables, int64_t T, const at::Device& dev, const char* op) {
  if (!row_seq.has_value()) {
    TORCH_CHECK_VALUE(tables.size(0) >= T, op, ": block_tables must have a row for each row of q (or row_seq says which)");
    return nullptr;
  }
  check_int(*row_seq, dev, at::kInt, op, "row_seq");
  TORCH_CHECK_VALUE(row_seq->numel() == T, op, ": row_seq must have a number for each row of q");
  return row_seq->data_ptr<int>();
}

void rope_cache_bounds(at::Tensor q_out, const at::Tensor& qkv, const at::Tensor& positions, const at::Tensor& cos_sin, int64_t nh,
                       int64_t nkv, int64_t hd, const at::Tensor& slots, at::Tensor k_cache, at::Tensor v_cache, at::Tensor bounds,
                       int64_t mode) {
  const char* op = "rope_cache_bounds";
  const at::Device dev = qkv.device();
  check_heads(nh, nkv, hd, op);
  check_rows(qkv, (nh + 2 * nkv) * hd, dev, op, "qkv");
  check_cache(k_cache, nkv, dev, op, "k_cache");
  check_cache(v_cache, nkv, dev, op, "v_cache");
  check_bounds(bounds, nkv, hd, dev, op);
  TORCH_CHECK_VALUE(k_cache.size(3) == hd && k_cache.sizes() == v_cache.sizes() && bounds.size(0) == k_cache.size(0), op,
                    ": k_cache, v_cache and bounds must have the same blocks and dims");
  const int64_t T = qkv.size(0);
  check_int(positions, dev, at::kInt, op, "positions");
  check_int(slots, dev, at::kInt, op, "slot_mapping");
  TORCH_CHECK_VALUE(positions.numel() == T && slots.numel() == T && T <= (1 << 29), op,
                    ": positions and slot_mapping must have a number for each row");
  TORCH_CHECK_VALUE(cos_sin.is_cuda() && cos_sin.device() == dev && cos_sin.scalar_type() == at::kFloat && cos_sin.is_contiguous() &&
                        cos_sin.dim() == 2 && cos_sin.size(0) > 0 && cos_sin.size(0) <= kInt && aligned(cos_sin),
                    op, ": cos_sin must be contiguous fp32 [positions, rotated dims]");
  const int64_t rd = cos_sin.size(1);
  TORCH_CHECK_VALUE(mode == 0 || mode == 1, op, ": mode is 0 (halves) or 1 (interleaved pairs)");
  TORCH_CHECK_VALUE(rd > 0 && rd <= hd && rd % (mode == 0 ? 16 : 8) == 0, op, ": rotated dims must be a multiple of ", mode == 0 ? 16 : 8,
                    " and at most the head's");
  check_rows(q_out, nh * hd, dev, op, "out");
  TORCH_CHECK_VALUE(q_out.is_contiguous() && q_out.size(0) == T && q_out.size(1) == nh * hd, op, ": out must be contiguous [rows, heads * dims]");
  const c10::DeviceGuard guard(dev);
  check_rc(dgi_rope_cache_bounds(qkv.data_ptr(), qkv.stride(0), (int)T, positions.data_ptr<int>(), (int)cos_sin.size(0),
                                 cos_sin.data_ptr<float>(), (int)nh, (int)nkv, (int)hd, (int)rd, (int)mode, slots.data_ptr<int>(),
                                 k_cache.size(0) * k_cache.size(2), q_out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                                 bounds.data_ptr(), (int)k_cache.size(2), cur_stream()), op);
}

void page_bounds(const at::Tensor& k_cache, at::Tensor bounds, const at::Tensor& pages, const at::Tensor& lens) {
  const char* op = "page_bounds";
  const at::Device dev = k_cache.device();
  TORCH_CHECK_VALUE(k_cache.dim() == 4, op, ": k_cache must be contiguous [blocks, kv heads, block size, dims]");
  const int64_t nkv = k_cache.size(1), hd = k_cache.size(3);
  check_cache(k_cache, nkv, dev, op, "k_cache");
  check_heads(nkv, nkv, hd, op);
  check_bounds(bounds, nkv, hd, dev, op);
  TORCH_CHECK_VALUE(bounds.size(0) == k_cache.size(0), op, ": bounds must have the cache's blocks");
  check_int(pages, dev, at::kInt, op, "pages");
  check_int(lens, dev, at::kInt, op, "lens");
  TORCH_CHECK_VALUE(pages.numel() == lens.numel() && pages.numel() <= kInt / nkv, op, ": pages and lens must be as many");
  const c10::DeviceGuard guard(dev);
  check_rc(dgi_page_bounds(k_cache.data_ptr(), bounds.data_ptr(), pages.data_ptr<int>(), lens.data_ptr<int>(), (int)pages.numel(),
                           (int)k_cache.size(0), (int)nkv, (int)hd, (int)k_cache.size(2), cur_stream()), op);
}

void select_pages(at::Tensor out, const at::Tensor& q, const at::Tensor& bounds, const at::Tensor& tables, const at::Tensor& ctx, int64_t nh,
                  int64_t nkv, int64_t page, int64_t first, int64_t recent, const c10::optional<at::Tensor>& row_seq) {
  const char* op = "select_pages";
  const at::Device dev = q.device();
  TORCH_CHECK_VALUE(bounds.dim() == 4, op, ": bounds must be contiguous [blocks, kv heads, 2, dims]");
  const int64_t hd = bounds.size(3);
  check_heads(nh, nkv, hd, op);
  check_rows(q, nh * hd, dev, op, "q");
  const int64_t T = q.size(0);
  check_bounds(bounds, nkv, hd, dev, op);
  check_tables(tables, dev, op);
  check_int(ctx, dev, at::kInt, op, "context_lens");
  TORCH_CHECK_VALUE(ctx.numel() == T, op, ": context_lens must have a number for each row of q");
  check_int(out, dev, at::kInt, op, "out");
  TORCH_CHECK_VALUE(out.dim() == 3 && out.size(0) == T && out.size(1) == nkv, op, ": out must be [rows, kv heads, count]");
  const int64_t count = out.size(2);
  TORCH_CHECK_VALUE(page > 0 && page <= (1 << 20), op, ": a page has 1 to 2^20 tokens");
  TORCH_CHECK_VALUE(first >= 0 && recent >= 1 && first + recent <= count, op, ": first >= 0, recent >= 1 and both within count");
  const int* rows = rows_of(row_seq, tables, T, dev, op);
  TORCH_CHECK_VALUE(T <= kInt / nkv && tables.size(1) <= (1 << 24), op, ": too many rows or pages");
  const c10::DeviceGuard guard(dev);
  // scores of as many rows at a time (by 16) as 256 MB hold
  const int64_t stride = tables.size(1), rows_16 = std::max<int64_t>((1 << 25) / (16 * nkv * std::max<int64_t>(stride, 1)), 1);
  const int64_t at_once = stride > count ? std::min(T, 16 * rows_16) : T;
  const at::Tensor keys = at::empty({stride > count ? at_once * nkv * stride : 0}, q.options().dtype(at::kLong));
  check_rc(dgi_select_pages(q.data_ptr(), q.stride(0), bounds.data_ptr(), tables.data_ptr<int>(), (int)tables.stride(0), (int)tables.size(1),
                            (int)tables.size(0), (int)bounds.size(0), ctx.data_ptr<int>(), rows, (int)T, (int)nh, (int)nkv, (int)hd,
                            (int)page, (int)count, (int)first, (int)recent, keys.data_ptr(), (int)stride, (int)at_once, out.data_ptr<int>(),
                            cur_stream()), op);
}

struct Attention {
  int64_t hd, page;
  at::Device dev;
};

Attention check_attention(const at::Tensor& out, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& tables,
                          int64_t nh, int64_t nkv, const char* op) {
  const at::Device dev = q.device();
  TORCH_CHECK_VALUE(k.dim() == 4, op, ": k_cache must be contiguous [blocks, kv heads, block size, dims]");
  const int64_t hd = k.size(3), page = k.size(2);
  check_heads(nh, nkv, hd, op);
  check_cache(k, nkv, dev, op, "k_cache");
  check_cache(v, nkv, dev, op, "v_cache");
  TORCH_CHECK_VALUE(k.sizes() == v.sizes(), op, ": k_cache and v_cache must be alike");
  TORCH_CHECK_VALUE((page & (page - 1)) == 0, op, ": pages of a power of two");
  check_rows(q, nh * hd, dev, op, "q");
  check_rows(out, nh * hd, dev, op, "out");
  TORCH_CHECK_VALUE(out.size(0) == q.size(0), op, ": out must have the rows of q");
  check_tables(tables, dev, op);
  TORCH_CHECK_VALUE(tables.size(1) <= (1 << 30) / page, op, ": a table has at most 2^30 tokens");
  return {hd, page, dev};
}

// Runs of `keys` for each of `units` workgroups, at most `most`: as many as give the card two workgroups a compute unit, but no more than
// 16, or 512 keys each, and 8 for `some` units and more: each is a part to be read again (8 rows of heads, 8192 keys: 16 runs 13.9 us, 32 15.0; 16,
// 8 runs 18.4, 32 22.2; trees of 4 nodes over 8000 keys, 8 heads: 16 runs 15.9, 62 22.6).
int64_t runs_of(int64_t units, int64_t keys, int64_t most, int64_t some) {
  return std::max<int64_t>(1, std::min<int64_t>({512 / std::max<int64_t>(1, units), most, units >= some ? 8 : std::max<int64_t>(16, keys / 512), 64}));
}

// What the parts of a split sum leave: a row of hd values each, and its logarithm.  Both in one tensor: allocating takes the host a
// microsecond, which a call of one row feels.
struct Parts {
  at::Tensor store;
  float *o = nullptr, *l = nullptr;

  Parts(int64_t n, int64_t hd, const at::Tensor& like) {
    if (n == 0) return;
    store = at::empty({n * (hd + 1)}, like.options().dtype(at::kFloat));
    o = store.data_ptr<float>();
    l = o + n * hd;
  }
};

void paged_selected(at::Tensor out, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& tables,
                    const at::Tensor& ctx, const at::Tensor& pages, int64_t nh, int64_t nkv, double scale,
                    const c10::optional<at::Tensor>& row_seq) {
  const char* op = "paged_selected";
  const Attention at_ = check_attention(out, q, k, v, tables, nh, nkv, op);
  const int64_t T = q.size(0);
  check_int(ctx, at_.dev, at::kInt, op, "context_lens");
  TORCH_CHECK_VALUE(ctx.numel() == T, op, ": context_lens must have a number for each row of q");
  check_int(pages, at_.dev, at::kInt, op, "pages");
  TORCH_CHECK_VALUE(pages.dim() == 3 && pages.size(0) == T && pages.size(1) == nkv && pages.size(2) > 0 && pages.size(2) <= (1 << 24), op,
                    ": pages must be [rows, kv heads, count]");
  const int* rows = rows_of(row_seq, tables, T, at_.dev, op);
  const int64_t count = pages.size(2);
  TORCH_CHECK_VALUE(T <= kInt / nkv - 16, op, ": too many rows");
  const c10::DeviceGuard guard(at_.dev);
  // Runs of 256 keys at the least, as many as give the card two workgroups a compute unit, where that is worth a second launch.  One run /
  // these, us, of 128 dims: 8 (row, head) pairs of 512 keys 8.6, 9.7, of 768 10.2, 9.8 (but one launch for the host), of 1024 11.7, 9.6, of 8192 58, 15; 64 of
  // 1024 12.6, 11.7, of 8192 73, 49; 96 of 1024 13.3, 16.5, of 4096 35.5, 39.3, of 8192 109, 86; 128 of 2048 25, 29.7, of 8192 125, 109; 192 160, 170.
  const int64_t least = std::max<int64_t>(1, 256 / at_.page), keys = count * at_.page, units = T * nkv;
  const bool one = keys < 1024 || (units > 64 && keys < 8192) || units > 160;
  const int64_t splits = one ? 1 : runs_of(units, keys, (count + least - 1) / least, 16);
  const Parts parts(splits > 1 ? T * nh * splits : 0, at_.hd, q);
  auto run = [&](int64_t t0, int64_t n, void* plan, int* plan_total, int* plan_rows) {
    const auto from = [&](const at::Tensor& t) { return static_cast<char*>(t.data_ptr()) + t0 * t.stride(0) * t.element_size(); };
    check_rc(dgi_paged_selected(from(q), q.stride(0), k.data_ptr(), v.data_ptr(), tables.data_ptr<int>(), (int)tables.stride(0),
                                (int)tables.size(1), (int)tables.size(0), (int)k.size(0), ctx.data_ptr<int>() + t0, rows ? rows + t0 : nullptr,
                                pages.data_ptr<int>() + t0 * nkv * count, (int)count, from(out), out.stride(0), parts.o, parts.l, (int)splits, plan,
                                plan_total, plan_rows, (int)n, (int)nh, (int)nkv, (int)at_.hd, (int)at_.page, (float)scale, cur_stream()), op);
  };
  // More rows than sequences, and enough of them to take the launch that makes the unions and still fill the card: neighbours read their
  // pages together, 16 / heads of a group at a time.  Each by itself / together, us, lists of 64 pages drawn at random, half alike, alike:
  // 128 rows of 32 heads on 8 of 128 dims 32, 40, 30, 19; 512 103, 91, 67, 41; 256 of 16 on 4 of 256 dims 86, 74, 54, 32, but 128 of them 44, 72, 53, 31;
  // two at a time, 256 rows of 28 on 4 31, 37, 33, 25; 512 57, 62, 54, 39; 2048 of 8 on one of 64 dims 31, 40, 36, 27.
  const int64_t side = 16 * nkv / nh;
  if (rows && T > tables.size(0) && side >= 2 && T * nkv * std::min<int64_t>(at_.hd, 128) >= (side >= 4 ? 1 : 2) * 131072) {
    // unions of as many rows at a time (by 16) as 256 MB hold
    const int64_t at_once = std::min(T, 16 * std::max<int64_t>((1 << 28) / (16 * nkv * count * 16), 1));
    const int64_t entries = at_once * nkv * count * 2, numbers = at_once * (nkv + 1);
    const at::Tensor plan = at::empty({entries + (numbers + 1) / 2}, q.options().dtype(at::kLong));
    int* plan_n = reinterpret_cast<int*>(plan.data_ptr<int64_t>() + entries);
    for (int64_t t0 = 0; t0 < T; t0 += at_once) run(t0, std::min(at_once, T - t0), plan.data_ptr(), plan_n, plan_n + at_once * nkv);
  } else {
    run(0, T, nullptr, nullptr, nullptr);
  }
}

void paged_tree(at::Tensor out, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& tables,
                const at::Tensor& cu, const at::Tensor& ctx, const at::Tensor& mask, int64_t nh, int64_t nkv, double scale,
                int64_t max_nodes) {
  const char* op = "paged_tree";
  const Attention at_ = check_attention(out, q, k, v, tables, nh, nkv, op);
  check_int(ctx, at_.dev, at::kInt, op, "context_lens");
  const int64_t S = ctx.numel();
  check_int(cu, at_.dev, at::kInt, op, "cu_seqlens_q");
  TORCH_CHECK_VALUE(cu.numel() == S + 1 && tables.size(0) >= S, op,
                    ": cu_seqlens_q must have one number more than context_lens, block_tables as many rows");
  check_int(mask, at_.dev, at::kLong, op, "tree_mask");
  TORCH_CHECK_VALUE(max_nodes >= 1 && max_nodes <= 64, op, ": trees of 1 to 64 nodes");
  TORCH_CHECK_VALUE(mask.dim() == 2 && mask.size(0) >= S && mask.size(1) >= max_nodes && mask.size(1) <= kInt, op,
                    ": tree_mask must be [sequences, nodes]");
  const c10::DeviceGuard guard(at_.dev);
  // Columns of 16 pairs a workgroup (tree_rows) or row tiles of 128 (tree_tiles): by the workgroups of the first and the keys that all of them
  // read, weighed by how full the tiles would be.  us of both, 32 heads on 8 of 128 dims: one sequence of 32 nodes, 300 keys 11.5, 18.2, 4000
  // 18.9, 21.1, of 64, 8000 keys 38.5, 35.3; 16 of 16, 1000 22.9, 35.9, 4000 59.9, 61.2; 64 heads: 8 of 16, 1000 22.9, 35.9, 4000 60.5,
  // 48.1; 32 of 32, 1000 136, 55; 14 heads on 2 of 64 dims: 8 of 64, 1000 15.4, 26.7, 4000 39.2, 34.0.  The tables were as wide as the contexts:
  // the host does not know these, and a wider table counts as its width.
  const int64_t G = nh / nkv, width = tables.size(1) * at_.page, pairs = max_nodes * G, cols = (pairs + 15) / 16, tiles = (pairs + 127) / 128;
  const int64_t few = S * nkv * cols;
  if (pairs > 32 && at_.hd <= 128 && !(few <= 1024 && few * (width + 100) * cols <= 6400000 * tiles)) {
    const int64_t least = 4;
    const int64_t shares = std::max<int64_t>(1, std::min<int64_t>(512 / nkv, (S * tiles * ((width + 63) / 64) + least - 1) / least));
    TORCH_CHECK_VALUE(S * tiles * nkv <= kInt, op, ": too many sequences");
    const Parts parts(shares > 1 ? shares * nkv * 2 * 128 : 0, at_.hd, q);
    check_rc(dgi_tree_tiles(q.data_ptr(), q.stride(0), k.data_ptr(), v.data_ptr(), tables.data_ptr<int>(), (int)tables.stride(0),
                            (int)tables.size(1), (int)S, (int)k.size(0), (int)q.size(0), cu.data_ptr<int>(), ctx.data_ptr<int>(),
                            mask.data_ptr(), (int)mask.stride(0), (int)max_nodes, out.data_ptr(), out.stride(0),
                            parts.o, parts.l, (int)shares, (int)least, (int)nh, (int)nkv, (int)at_.hd, (int)at_.page, (float)scale,
                            cur_stream()), op);
    return;
  }
  TORCH_CHECK_VALUE(S <= kInt / 64 / (nkv * cols), op, ": too many sequences");
  // One run / several, us, 32 heads on 8 of 128 dims: a tree of 4 nodes, 300 keys 10.6, 11.2, 600 13.0, 11.4; 4 of 24 nodes, 300 11.1, 14.2, 1000
  // 17.5, 19.0; 16 of 4, 300 10.6, 12.7, 1000 17.7, 21.8; 8 of 8, 2000 26.3, 22.9; 16 of 8, 1000 18.5, 23.6, 4000 46, 52.
  const int64_t items = few, min_part = 128;
  const bool one = width <= 400 || (items >= 64 && width <= 10 * items) || items >= 224;
  const int64_t splits = one ? 1 : runs_of(items, width, (width + min_part - 1) / min_part, 32);
  const Parts parts(splits > 1 ? items * splits * 16 : 0, at_.hd, q);
  check_rc(dgi_tree_rows(q.data_ptr(), q.stride(0), k.data_ptr(), v.data_ptr(), tables.data_ptr<int>(), (int)tables.stride(0),
                          (int)tables.size(1), (int)S, (int)k.size(0), (int)q.size(0), cu.data_ptr<int>(), ctx.data_ptr<int>(),
                          mask.data_ptr(), (int)mask.stride(0), (int)max_nodes, out.data_ptr(), out.stride(0),
                          parts.o, parts.l, (int)splits, (int)min_part, (int)nh, (int)nkv, (int)at_.hd, (int)at_.page, (float)scale,
                          cur_stream()), op);
}

// The same with an output of the call's own: allocated here, a microsecond of the host's time that the smallest calls feel is half of what it
// takes from Python.
at::Tensor new_rows(const at::Tensor& q, int64_t cols, const char* op) {
  TORCH_CHECK_VALUE(q.dim() == 2 && cols >= 0 && cols <= kInt, op, ": rows of heads are two-dimensional");
  return at::empty({q.size(0), cols}, q.options());
}

at::Tensor rope_cache_bounds_new(const at::Tensor& qkv, const at::Tensor& positions, const at::Tensor& cos_sin, int64_t nh, int64_t nkv, int64_t hd,
                                 const at::Tensor& slots, at::Tensor k_cache, at::Tensor v_cache, at::Tensor bounds, int64_t mode) {
  check_heads(nh, nkv, hd, "rope_cache_bounds");
  at::Tensor out = new_rows(qkv, nh * hd, "rope_cache_bounds");
  rope_cache_bounds(out, qkv, positions, cos_sin, nh, nkv, hd, slots, k_cache, v_cache, bounds, mode);
  return out;
}

at::Tensor select_pages_new(const at::Tensor& q, const at::Tensor& bounds, const at::Tensor& tables, const at::Tensor& ctx, int64_t nh, int64_t nkv,
                            int64_t page, int64_t count, int64_t first, int64_t recent, const c10::optional<at::Tensor>& row_seq) {
  TORCH_CHECK_VALUE(q.dim() == 2 && nkv > 0 && count > 0 && count <= kInt, "select_pages: rows of heads, kv heads and pages to keep");
  at::Tensor out = at::empty({q.size(0), nkv, count}, q.options().dtype(at::kInt));
  select_pages(out, q, bounds, tables, ctx, nh, nkv, page, first, recent, row_seq);
  return out;
}

at::Tensor paged_selected_new(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& tables, const at::Tensor& ctx,
                              const at::Tensor& pages, int64_t nh, int64_t nkv, double scale, const c10::optional<at::Tensor>& row_seq) {
  TORCH_CHECK_VALUE(k.dim() == 4, "paged_selected: k_cache must be contiguous [blocks, kv heads, block size, dims]");
  check_heads(nh, nkv, k.size(3), "paged_selected");
  at::Tensor out = new_rows(q, nh * k.size(3), "paged_selected");
  paged_selected(out, q, k, v, tables, ctx, pages, nh, nkv, scale, row_seq);
  return out;
}

at::Tensor paged_tree_new(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& tables, const at::Tensor& cu,
                          const at::Tensor& ctx, const at::Tensor& mask, int64_t nh, int64_t nkv, double scale, int64_t max_nodes) {
  TORCH_CHECK_VALUE(k.dim() == 4, "paged_tree: k_cache must be contiguous [blocks, kv heads, block size, dims]");
  check_heads(nh, nkv, k.size(3), "paged_tree");
  at::Tensor out = new_rows(q, nh * k.size(3), "paged_tree");
  paged_tree(out, q, k, v, tables, cu, ctx, mask, nh, nkv, scale, max_nodes);
  return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(dgi, m) {
  m.def("rope_cache_bounds(Tensor(a!) out, Tensor qkv, Tensor positions, Tensor cos_sin, int nh, int nkv, int hd, Tensor slot_mapping, "
        "Tensor(b!) k_cache, Tensor(c!) v_cache, Tensor(d!) bounds, int mode) -> ()");
  m.def("page_bounds(Tensor k_cache, Tensor(a!) bounds, Tensor pages, Tensor lens) -> ()");
  m.def("select_pages(Tensor(a!) out, Tensor q, Tensor bounds, Tensor block_tables, Tensor context_lens, int nh, int nkv, int page, int first, "
        "int recent, Tensor? row_seq) -> ()");
  m.def("paged_selected(Tensor(a!) out, Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_tables, Tensor context_lens, Tensor pages, "
        "int nh, int nkv, float scale, Tensor? row_seq) -> ()");
  m.def("paged_tree(Tensor(a!) out, Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_tables, Tensor cu_seqlens_q, Tensor context_lens, "
        "Tensor tree_mask, int nh, int nkv, float scale, int max_nodes) -> ()");
  m.def("rope_cache_bounds_new(Tensor qkv, Tensor positions, Tensor cos_sin, int nh, int nkv, int hd, Tensor slot_mapping, Tensor(a!) k_cache, "
        "Tensor(b!) v_cache, Tensor(c!) bounds, int mode) -> Tensor");
  m.def("select_pages_new(Tensor q, Tensor bounds, Tensor block_tables, Tensor context_lens, int nh, int nkv, int page, int count, int first, "
        "int recent, Tensor? row_seq) -> Tensor");
  m.def("paged_selected_new(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_tables, Tensor context_lens, Tensor pages, int nh, int nkv, "
        "float scale, Tensor? row_seq) -> Tensor");
  m.def("paged_tree_new(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_tables, Tensor cu_seqlens_q, Tensor context_lens, "
        "Tensor tree_mask, int nh, int nkv, float scale, int max_nodes) -> Tensor");
}

TORCH_LIBRARY_IMPL(dgi, CUDA, m) {
  m.impl("rope_cache_bounds", &rope_cache_bounds);
  m.impl("page_bounds", &page_bounds);
  m.impl("select_pages", &select_pages);
  m.impl("paged_selected", &paged_selected);
  m.impl("paged_tree", &paged_tree);
  m.impl("rope_cache_bounds_new", &rope_cache_bounds_new);
  m.impl("select_pages_new", &select_pages_new);
  m.impl("paged_selected_new", &paged_selected_new);
  m.impl("paged_tree_new", &paged_tree_new);
}
