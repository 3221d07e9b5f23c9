// Torch bindings of the paged KV cache (include/megaqwen_b200.h, "paged KV
// cache"): argument checks that raise RuntimeError, outputs and workspaces from
// the caching allocator on the current stream.  The reference has no
// counterpart; Python names are in megaqwen_b200/paged.py.

#include <torch/extension.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>
#include <stdexcept>
#include <string>
#include <tuple>

#include "megaqwen_b200.h"

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

[[noreturn]] void fail(const std::string& what) { throw std::runtime_error(what); }

void raise_rc(int rc, const char* where) {
    if (rc)
        fail(std::string(where) + ": " + mq_error_string(rc) + " (code " + std::to_string(rc) + ")" +
             (rc == MQ_ERR_CUDA ? std::string(" ") + mq_last_error_detail() : ""));
}

// Uninitialised tensors straight from the caching allocator: the dispatcher's
// path costs about half of a short call's host time.
Tensor blank(at::IntArrayRef sizes, torch::ScalarType type, const torch::Device& dev) {
    return Tensor(at::detail::empty_cuda(sizes, type, dev, c10::nullopt));
}
Tensor scratch(size_t bytes, const torch::Device& dev) { return blank({(int64_t)bytes}, torch::kUInt8, dev); }

cudaStream_t stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

int dtype_of(const Tensor& t, const char* name) {
    if (t.scalar_type() == torch::kBFloat16) return MQ_BF16;
    if (t.scalar_type() == torch::kHalf) return MQ_FP16;
    fail(std::string(name) + " must be bfloat16 or float16");
}

void on(const Tensor& t, const torch::Device& dev, const char* name) {
    if (t.device() != dev) fail(std::string(name) + " must be on " + dev.str());
}

// 1-D contiguous int32 on `dev`
int* ints(const Tensor& t, const torch::Device& dev, const char* name, int64_t n = -1) {
    on(t, dev, name);
    if (t.scalar_type() != torch::kInt32 || t.dim() != 1 || !t.is_contiguous())
        fail(std::string(name) + " must be a contiguous 1-D int32 tensor");
    if (n >= 0 && t.numel() != n) fail(std::string(name) + " must have " + std::to_string(n) + " entries");
    if (t.numel() > 0x7fffffffll) fail(std::string(name) + " is too long");
    return t.data_ptr<int>();
}

int* status_of(const OptTensor& s, const torch::Device& dev) {
    return s.has_value() ? ints(*s, dev, "status", 1) : nullptr;
}

mq_paged_pool pool_of(const Tensor& k, const Tensor& v, const OptTensor& index) {
    if (!k.is_cuda()) fail("k_pages must be a CUDA tensor");
    mq_paged_pool p = {};
    p.dtype = dtype_of(k, "k_pages");
    if (k.dim() != 5 || v.sizes() != k.sizes() || v.scalar_type() != k.scalar_type())
        fail("k_pages and v_pages must both be [pages, layers, kv_heads, page_size, head_dim] of one type");
    on(v, k.device(), "v_pages");
    const int64_t D = k.size(4), page = k.size(3);
    if (D != 64 && D != 128) fail("head_dim must be 64 or 128");
    if (page != 16 && page != 32 && page != 64 && page != 128) fail("page_size must be 16, 32, 64 or 128");
    for (int i = 0; i < 3; ++i)
        if (k.size(i) < 1 || k.size(i) > 0x7fffffff) fail("k_pages has an empty or too long dimension");
    if (k.stride(4) != 1 || k.stride(3) != D || v.stride(4) != 1 || v.stride(3) != D)
        fail("the [page_size, head_dim] blocks of k_pages and v_pages must be contiguous");
    p.k = k.data_ptr();
    p.v = v.data_ptr();
    p.num_pages = (int)k.size(0);
    p.num_layers = (int)k.size(1);
    p.num_kv_heads = (int)k.size(2);
    p.page_size = (int)page;
    p.head_dim = (int)D;
    p.k_page = k.stride(0); p.k_layer = k.stride(1); p.k_head = k.stride(2);
    p.v_page = v.stride(0); p.v_layer = v.stride(1); p.v_head = v.stride(2);
    if (index.has_value()) {
        const Tensor& x = *index;
        on(x, k.device(), "index");
        if (x.scalar_type() != torch::kInt8 || x.dim() != 4 || x.size(0) != k.size(0) || x.size(1) != k.size(1) ||
            x.size(2) != k.size(2) || x.size(3) != 2 * D + 16 || x.stride(3) != 1)
            fail("index must be int8 [pages, layers, kv_heads, 2 * head_dim + 16]");
        p.index = (signed char*)x.data_ptr();
        p.i_page = x.stride(0); p.i_layer = x.stride(1); p.i_head = x.stride(2);
    }
    const auto odd = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) != 0; };
    if (odd(p.k) || odd(p.v) || odd(p.index) ||
        (p.k_page | p.k_layer | p.k_head | p.v_page | p.v_layer | p.v_head) % 8 || (p.i_page | p.i_layer | p.i_head) % 16)
        fail("k_pages, v_pages and index must be aligned to 16 bytes, strides included");
    return p;
}

void table_ok(const Tensor& t, const torch::Device& dev) {
    on(t, dev, "page_table");
    if (t.scalar_type() != torch::kInt32 || t.dim() != 2 || t.size(0) < 1 || t.size(1) < 1 ||
        (t.size(1) > 1 && t.stride(1) != 1) || (t.size(0) > 1 && t.stride(0) < t.size(1)))
        fail("page_table must be int32 [slots, pages per slot] with contiguous rows");
    if (t.size(0) > 0x7fffffffll || t.size(1) > 0x7fffffffll) fail("page_table is too large");
}
long long row_of(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

struct Table {
    mq_page_table c = {};
    Tensor ws;
    Table(const Tensor& table, const OptTensor& lengths, const Tensor& refs, int64_t page_size, int64_t n,
          const OptTensor& status, bool workspace) {
        if (!table.is_cuda()) fail("page_table must be a CUDA tensor");
        const auto dev = table.device();
        table_ok(table, dev);
        if (table.size(0) > 65536) fail("page_table has more than 65536 slots");
        if (n > table.size(0)) fail("more slots named than the page table has");
        if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128)
            fail("page_size must be 16, 32, 64 or 128");
        c.table = table.data_ptr<int>();
        c.row_stride = row_of(table);
        c.num_slots = (int)table.size(0);
        c.cols = (int)table.size(1);
        c.lengths = lengths.has_value() ? ints(*lengths, dev, "lengths", table.size(0)) : nullptr;
        c.refs = ints(refs, dev, "refs");
        if (refs.numel() < 1 || refs.numel() > (1 << 20)) fail("refs must have between 1 and 2^20 pages");
        c.num_pages = (int)refs.numel();
        c.page_size = (int)page_size;
        c.status = status_of(status, dev);
        if (workspace) {
            c.workspace_bytes = mq_paged_workspace_bytes(c.num_pages, (int)n);
            ws = scratch(c.workspace_bytes, dev);
            c.workspace = ws.data_ptr();
        }
    }
};

void paged_free(Tensor table, Tensor lengths, Tensor refs, Tensor slots, int64_t page_size, OptTensor status) {
    Table t(table, lengths, refs, page_size, slots.numel(), status, false);
    c10::cuda::CUDAGuard guard(table.device());
    raise_rc(mq_paged_free(&t.c, ints(slots, table.device(), "slots"), (int)slots.numel(), stream_of(table)), "paged free");
}

void paged_reserve(Tensor table, Tensor lengths, Tensor refs, Tensor slots, Tensor new_lengths, int64_t page_size,
                   OptTensor status) {
    if (table.is_cuda()) ints(new_lengths, table.device(), "new_lengths", slots.numel());
    c10::cuda::OptionalCUDAGuard guard;
    if (table.is_cuda()) guard.set_device(table.device());
    Table t(table, lengths, refs, page_size, slots.numel(), status, true);
    raise_rc(mq_paged_reserve(&t.c, ints(slots, table.device(), "slots"), new_lengths.data_ptr<int>(), (int)slots.numel(),
                              stream_of(table)), "paged reserve");
}

void paged_fork(Tensor k, Tensor v, Tensor table, Tensor lengths, Tensor refs, Tensor parents, Tensor children,
                OptTensor status) {
    const mq_paged_pool pool = pool_of(k, v, c10::nullopt);
    on(table, k.device(), "page_table");
    c10::cuda::CUDAGuard guard(k.device());
    Table t(table, lengths, refs, pool.page_size, children.numel(), status, true);
    if (refs.numel() != k.size(0)) fail("refs must have one entry per page");
    raise_rc(mq_paged_fork(&pool, &t.c, ints(parents, k.device(), "parents", children.numel()),
                           ints(children, k.device(), "children"), (int)children.numel(), stream_of(k)), "paged fork");
}

std::tuple<Tensor, Tensor, Tensor> paged_accept(Tensor k, Tensor v, Tensor table, Tensor lengths, Tensor refs, Tensor slots,
                                                Tensor parents, Tensor tokens, Tensor chosen, OptTensor q_starts,
                                                OptTensor index, OptTensor status) {
    const mq_paged_pool pool = pool_of(k, v, index);
    const auto dev = k.device();
    on(table, dev, "page_table");
    const int* s = ints(slots, dev, "slots");
    const int n = (int)slots.numel();
    const int* up = ints(parents, dev, "parents");
    const int total = (int)parents.numel();
    const int* tok = ints(tokens, dev, "tokens", total);
    const int* at = ints(chosen, dev, "chosen", total);
    const int* starts = nullptr;
    if (q_starts.has_value()) starts = ints(*q_starts, dev, "q_starts", n + 1ll);
    else if (n != total) fail("without q_starts, a sequence must have one node");
    if (total && !n) fail("nodes without sequences");
    c10::cuda::CUDAGuard guard(dev);
    Table t(table, lengths, refs, pool.page_size, n, status, false);
    if (refs.numel() != k.size(0)) fail("refs must have one entry per page");
    Tensor path = blank({total}, torch::kInt32, dev), emitted = blank({total}, torch::kInt32, dev),
           count = blank({n}, torch::kInt32, dev);
    t.c.workspace_bytes = mq_paged_accept_workspace_bytes(total);
    t.ws = scratch(t.c.workspace_bytes, dev);
    t.c.workspace = t.ws.data_ptr();
    raise_rc(mq_paged_accept(&pool, &t.c, s, starts, up, tok, at, n, total, path.data_ptr<int>(), emitted.data_ptr<int>(),
                             count.data_ptr<int>(), stream_of(k)), "paged accept");
    return std::make_tuple(path, emitted, count);
}

void same_pools(const mq_paged_pool& a, const mq_paged_pool& b) {
    if (a.dtype != b.dtype || a.num_layers != b.num_layers || a.num_kv_heads != b.num_kv_heads ||
        a.page_size != b.page_size || a.head_dim != b.head_dim)
        fail("the two pools must have the same type, layers, kv heads, page size and head dim");
    if (!a.index != !b.index) fail("either both pools have an index or neither");
}

void paged_copy(Tensor k, Tensor v, Tensor src, Tensor dst, OptTensor dst_k, OptTensor dst_v, OptTensor index,
                OptTensor dst_index, OptTensor status) {
    const mq_paged_pool a = pool_of(k, v, index);
    if (dst_k.has_value() != dst_v.has_value()) fail("dst_k_pages and dst_v_pages go together");
    const mq_paged_pool b = dst_k.has_value() ? pool_of(*dst_k, *dst_v, dst_index) : a;
    if (dst_k.has_value()) on(*dst_k, k.device(), "dst_k_pages");
    same_pools(a, b);
    const int n = (int)src.numel();
    c10::cuda::CUDAGuard guard(k.device());
    Tensor ws = scratch(mq_paged_workspace_bytes(b.num_pages, n), k.device());
    raise_rc(mq_paged_copy(&a, &b, ints(src, k.device(), "src"), ints(dst, k.device(), "dst", n), n,
                           status_of(status, k.device()), ws.data_ptr(), (size_t)ws.numel(), stream_of(k)), "paged copy");
}

void paged_compact(Tensor k, Tensor v, Tensor table, Tensor refs, Tensor out_k, Tensor out_v, Tensor out_table,
                   Tensor out_refs, OptTensor index, OptTensor out_index, OptTensor status) {
    const mq_paged_pool a = pool_of(k, v, index), b = pool_of(out_k, out_v, out_index);
    on(out_k, k.device(), "out_k_pages");
    on(table, k.device(), "page_table");
    same_pools(a, b);
    if (a.k == b.k || a.v == b.v) fail("compact needs another pool to write to");
    c10::cuda::CUDAGuard guard(k.device());
    Table t(table, c10::nullopt, refs, a.page_size, 0, status, true);
    if (refs.numel() != k.size(0)) fail("refs must have one entry per page");
    table_ok(out_table, k.device());
    if (out_table.sizes() != table.sizes()) fail("out_table must have page_table's shape");
    if (out_table.data_ptr() == table.data_ptr() || out_refs.data_ptr() == refs.data_ptr())
        fail("compact needs tables of its own to write to");
    raise_rc(mq_paged_compact(&a, &b, &t.c, out_table.data_ptr<int>(), row_of(out_table),
                              ints(out_refs, k.device(), "out_refs", out_k.size(0)), stream_of(k)), "paged compact");
}

void heads(const Tensor& x, const char* name, int64_t n, int64_t D, const Tensor& like) {
    on(x, like.device(), name);
    if (x.dim() != 3 || x.size(2) != D || x.stride(2) != 1 || x.scalar_type() != like.scalar_type() || (n >= 0 && x.size(0) != n))
        fail(std::string(name) + " must be [tokens, heads, head_dim] of the cache's type, head_dim contiguous");
}

void rope_args(mq_rope_params& p, const Tensor& cos, const Tensor& sin, const torch::Device& dev, int64_t D,
               bool interleaved, bool inverse) {
    on(cos, dev, "cos");
    if (cos.scalar_type() != torch::kFloat32 || cos.dim() != 2 || sin.scalar_type() != torch::kFloat32 ||
        sin.sizes() != cos.sizes() || (cos.size(1) > 1 && (cos.stride(1) != 1 || sin.stride(1) != 1)))
        fail("cos and sin must be float32 [positions, rotary_dim / 2]");
    on(sin, dev, "sin");
    if (cos.size(0) < 1 || cos.size(1) * 2 > D) fail("rotary_dim must not exceed head_dim");
    p.cos_table = cos.data_ptr<float>();
    p.sin_table = sin.data_ptr<float>();
    p.cos_row = cos.stride(0);
    p.sin_row = sin.stride(0);
    p.max_pos = (int)std::min<int64_t>(cos.size(0), 0x7fffffff);
    p.rotary_dim = (int)cos.size(1) * 2;
    p.interleaved = interleaved;
    p.inverse = inverse;
}

Tensor rope(Tensor x, Tensor positions, Tensor cos, Tensor sin, bool interleaved, bool inverse, OptTensor status) {
    if (!x.is_cuda()) fail("x must be a CUDA tensor");
    mq_rope_params p = {};
    p.dtype = dtype_of(x, "x");
    if (x.dim() != 3 || (x.size(2) != 64 && x.size(2) != 128) || x.stride(2) != 1)
        fail("x must be [tokens, heads, head_dim] with head_dim 64 or 128 contiguous");
    const auto dev = x.device();
    rope_args(p, cos, sin, dev, x.size(2), interleaved, inverse);
    c10::cuda::CUDAGuard guard(dev);
    Tensor out = blank(x.sizes(), x.scalar_type(), dev);
    p.positions = ints(positions, dev, "positions", x.size(0));
    p.q = x.data_ptr();
    p.q_out = out.data_ptr();
    p.q_token = x.stride(0); p.q_head = x.stride(1);
    p.out_token = out.stride(0); p.out_head = out.stride(1);
    p.n = (int)x.size(0);
    p.num_q_heads = (int)x.size(1);
    p.head_dim = (int)x.size(2);
    p.status = status_of(status, dev);
    if (out.numel()) raise_rc(mq_rope(&p, stream_of(x)), "rope");
    return out;
}

Tensor rope_append(Tensor q, Tensor k, Tensor v, Tensor k_pages, Tensor v_pages, Tensor table, Tensor slots,
                   Tensor positions, Tensor cos, Tensor sin, int64_t layer, bool interleaved, OptTensor index,
                   OptTensor status, OptTensor places) {
    const mq_paged_pool pool = pool_of(k_pages, v_pages, index);
    const auto dev = k_pages.device();
    const int64_t D = pool.head_dim, n = q.dim() == 3 ? q.size(0) : -1;
    heads(q, "q", -1, D, k_pages);
    heads(k, "k", n, D, k_pages);
    heads(v, "v", n, D, k_pages);
    if (k.size(1) != pool.num_kv_heads || v.size(1) != pool.num_kv_heads) fail("k and v must have the cache's kv heads");
    if (layer < 0 || layer >= pool.num_layers) fail("layer out of range");
    table_ok(table, dev);
    mq_rope_params p = {};
    rope_args(p, cos, sin, dev, D, interleaved, false);
    c10::cuda::CUDAGuard guard(dev);
    Tensor out = blank(q.sizes(), q.scalar_type(), dev);
    p.dtype = pool.dtype;
    p.q = q.data_ptr();
    p.q_out = out.data_ptr();
    p.k = k.data_ptr();
    p.v = v.data_ptr();
    p.q_token = q.stride(0); p.q_head = q.stride(1);
    p.out_token = out.stride(0); p.out_head = out.stride(1);
    p.k_token = k.stride(0); p.k_head = k.stride(1);
    p.v_token = v.stride(0); p.v_head = v.stride(1);
    p.positions = ints(positions, dev, "positions", n);
    p.slots = ints(slots, dev, "slots", n);
    if (places.has_value()) p.places = ints(*places, dev, "places", n);
    p.n = (int)n;
    p.num_q_heads = (int)q.size(1);
    p.head_dim = (int)D;
    p.layer = (int)layer;
    p.pool = &pool;
    p.table = table.data_ptr<int>();
    p.table_row = row_of(table);
    p.num_slots = (int)table.size(0);
    p.table_cols = (int)table.size(1);
    p.status = status_of(status, dev);
    raise_rc(mq_rope(&p, stream_of(q)), "rope_append");
    return out;
}

// q as the kernels read it: 16-byte pieces of a head row (a contiguous q may start anywhere, so a copy and not
// contiguous(), which would hand it back)
Tensor pieces(const Tensor& q) {
    const bool ok = (reinterpret_cast<uintptr_t>(q.data_ptr()) & 15) == 0 && q.stride(0) % 8 == 0 && q.stride(1) % 8 == 0;
    return ok ? q : q.clone(at::MemoryFormat::Contiguous);
}

int q_heads(const Tensor& q, const mq_paged_pool& pool) {
    if (q.size(1) < 1 || q.size(1) % pool.num_kv_heads) fail("q heads must be a multiple of the kv heads");
    return (int)q.size(1);
}

Tensor attend(Tensor q, Tensor k_pages, Tensor v_pages, Tensor table, Tensor lengths, Tensor slots, int64_t layer,
              OptTensor q_starts, OptTensor group_starts, OptTensor prefix_pages, c10::optional<double> scale,
              OptTensor status) {
    const mq_paged_pool pool = pool_of(k_pages, v_pages, c10::nullopt);
    const auto dev = k_pages.device();
    heads(q, "q", -1, pool.head_dim, k_pages);
    table_ok(table, dev);
    if (layer < 0 || layer >= pool.num_layers) fail("layer out of range");
    mq_paged_attend_params p = {};
    p.num_q_heads = q_heads(q, pool);
    p.slots = ints(slots, dev, "slots");
    if (slots.numel() > 2048) fail("at most 2048 sequences per call");
    p.num_seqs = (int)slots.numel();
    p.total_q = (int)q.size(0);
    if (q_starts.has_value()) p.q_starts = ints(*q_starts, dev, "q_starts", slots.numel() + 1);
    else if (q.size(0) != slots.numel()) fail("without q_starts, q must have one token per sequence");
    if (group_starts.has_value() != prefix_pages.has_value()) fail("group_starts and prefix_pages go together");
    if (group_starts.has_value()) {
        p.group_starts = ints(*group_starts, dev, "group_starts");
        if (group_starts->numel() < 1) fail("group_starts must have one entry more than there are groups");
        p.num_groups = (int)group_starts->numel() - 1;
        if (p.num_groups > p.num_seqs) fail("more groups than sequences");
        p.prefix_pages = ints(*prefix_pages, dev, "prefix_pages", p.num_groups);
    }
    if (q.size(0) && !slots.numel()) fail("query tokens without sequences");
    c10::cuda::CUDAGuard guard(dev);
    const Tensor qq = pieces(q);
    Tensor out = blank(q.sizes(), q.scalar_type(), dev);
    if (!out.numel()) return out;
    p.pool = &pool;
    p.q = qq.data_ptr();
    p.q_token = qq.stride(0);
    p.q_head = qq.stride(1);
    p.out = out.data_ptr();
    p.table = table.data_ptr<int>();
    p.table_row = row_of(table);
    p.num_slots = (int)table.size(0);
    p.table_cols = (int)table.size(1);
    p.lengths = ints(lengths, dev, "lengths", table.size(0));
    p.layer = (int)layer;
    p.scale = scale.has_value() ? (float)*scale : 1.0f / std::sqrt((float)pool.head_dim);
    p.status = status_of(status, dev);
    p.workspace_bytes = mq_paged_attend_workspace_bytes(&p);
    Tensor ws = scratch(p.workspace_bytes, dev);
    p.workspace = ws.data_ptr();
    raise_rc(mq_paged_attend(&p, stream_of(q)), "attend");
    return out;
}

// The part that window_attend and tree_attend share; run(params, stream) makes the call.
template <typename Run>
Tensor span_attend(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& table, const Tensor& lengths,
                   const Tensor& slots, int64_t layer, const OptTensor& q_starts, c10::optional<double> scale,
                   const OptTensor& status, const char* name, Run run) {
    const mq_paged_pool pool = pool_of(k_pages, v_pages, c10::nullopt);
    const auto dev = k_pages.device();
    heads(q, "q", -1, pool.head_dim, k_pages);
    table_ok(table, dev);
    if (layer < 0 || layer >= pool.num_layers) fail("layer out of range");
    mq_paged_span_params p = {};
    p.num_q_heads = q_heads(q, pool);
    p.slots = ints(slots, dev, "slots");
    if (slots.numel() > 2048) fail("at most 2048 sequences per call");
    p.num_seqs = (int)slots.numel();
    if (q.size(0) > 0x7fffffffll) fail("too many query tokens");
    p.total_q = (int)q.size(0);
    if (q_starts.has_value()) p.q_starts = ints(*q_starts, dev, "q_starts", slots.numel() + 1);
    else if (q.size(0) != slots.numel()) fail("without q_starts, q must have one token per sequence");
    if (q.size(0) && !slots.numel()) fail("query tokens without sequences");
    p.lengths = ints(lengths, dev, "lengths", table.size(0));
    p.status = status_of(status, dev);
    c10::cuda::CUDAGuard guard(dev);
    const Tensor qq = pieces(q);
    Tensor out = blank(q.sizes(), q.scalar_type(), dev);
    if (!out.numel()) return out;
    p.pool = &pool;
    p.q = qq.data_ptr();
    p.q_token = qq.stride(0);
    p.q_head = qq.stride(1);
    p.out = out.data_ptr();
    p.table = table.data_ptr<int>();
    p.table_row = row_of(table);
    p.num_slots = (int)table.size(0);
    p.table_cols = (int)table.size(1);
    p.layer = (int)layer;
    p.scale = scale.has_value() ? (float)*scale : 1.0f / std::sqrt((float)pool.head_dim);
    p.workspace_bytes = mq_paged_span_workspace_bytes(&p);
    Tensor ws = scratch(p.workspace_bytes, dev);
    p.workspace = ws.data_ptr();
    raise_rc(run(&p, stream_of(q)), name);
    return out;
}

Tensor window_attend(Tensor q, Tensor k_pages, Tensor v_pages, Tensor table, Tensor lengths, Tensor slots, int64_t layer,
                     int64_t window, int64_t sinks, OptTensor q_starts, c10::optional<double> scale, OptTensor status) {
    if (window < 1) fail("window must be positive");
    if (sinks < 0) fail("sinks must not be negative");
    const int w = (int)std::min<int64_t>(window, 0x7fffffff), n = (int)std::min<int64_t>(sinks, 0x7fffffff);
    return span_attend(q, k_pages, v_pages, table, lengths, slots, layer, q_starts, scale, status, "window_attend",
                       [&](const mq_paged_span_params* p, cudaStream_t st) { return mq_paged_window(p, w, n, st); });
}

Tensor tree_attend(Tensor q, Tensor k_pages, Tensor v_pages, Tensor table, Tensor lengths, Tensor slots, Tensor parents,
                   int64_t layer, OptTensor q_starts, c10::optional<double> scale, OptTensor status) {
    if (!k_pages.is_cuda()) fail("k_pages must be a CUDA tensor");
    const int* up = ints(parents, k_pages.device(), "parents", q.dim() == 3 ? q.size(0) : -1);
    return span_attend(q, k_pages, v_pages, table, lengths, slots, layer, q_starts, scale, status, "tree_attend",
                       [&](const mq_paged_span_params* p, cudaStream_t st) { return mq_paged_tree(p, up, st); });
}

std::tuple<Tensor, Tensor> sparse_attend(Tensor q, Tensor k_pages, Tensor v_pages, Tensor index, Tensor table,
                                         Tensor slots, Tensor positions, int64_t layer, int64_t top_k,
                                         c10::optional<double> scale, OptTensor status) {
    const mq_paged_pool pool = pool_of(k_pages, v_pages, index);
    const auto dev = k_pages.device();
    heads(q, "q", -1, pool.head_dim, k_pages);
    table_ok(table, dev);
    if (layer < 0 || layer >= pool.num_layers) fail("layer out of range");
    if (top_k < 1 || top_k > 49152) fail("top_k must be between 1 and 49152");
    if (table.size(1) > 49152) fail("sparse attention takes at most 49152 pages per slot");
    mq_paged_sparse_params p = {};
    p.num_q_heads = q_heads(q, pool);
    if (p.num_q_heads / pool.num_kv_heads > 64) fail("at most 64 q heads per kv head");
    p.n = (int)q.size(0);
    p.slots = ints(slots, dev, "slots", q.size(0));
    p.positions = ints(positions, dev, "positions", q.size(0));
    c10::cuda::CUDAGuard guard(dev);
    const Tensor qq = pieces(q);
    Tensor out = blank(q.sizes(), q.scalar_type(), dev);
    Tensor sel = blank({q.size(0), pool.num_kv_heads, top_k}, torch::kInt32, dev);
    if (!out.numel()) return std::make_tuple(out, sel);
    p.pool = &pool;
    p.q = qq.data_ptr();
    p.q_token = qq.stride(0);
    p.q_head = qq.stride(1);
    p.out = out.data_ptr();
    p.selected = sel.data_ptr<int>();
    p.table = table.data_ptr<int>();
    p.table_row = row_of(table);
    p.num_slots = (int)table.size(0);
    p.table_cols = (int)table.size(1);
    p.layer = (int)layer;
    p.top_k = (int)top_k;
    p.scale = scale.has_value() ? (float)*scale : 1.0f / std::sqrt((float)pool.head_dim);
    p.status = status_of(status, dev);
    p.workspace_bytes = mq_paged_sparse_workspace_bytes(&p);
    Tensor ws = scratch(p.workspace_bytes, dev);
    p.workspace = ws.data_ptr();
    raise_rc(mq_paged_sparse(&p, stream_of(q)), "sparse_attend");
    return std::make_tuple(out, sel);
}

}  // namespace

void bind_paged(py::module_& m) {
    const auto none = py::none();
    m.def("paged_rope", &rope, py::arg("x"), py::arg("positions"), py::arg("cos"), py::arg("sin"),
          py::arg("interleaved") = false, py::arg("inverse") = false, py::arg("status") = none);
    m.def("paged_rope_append", &rope_append, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("k_pages"),
          py::arg("v_pages"), py::arg("page_table"), py::arg("slots"), py::arg("positions"), py::arg("cos"),
          py::arg("sin"), py::arg("layer"), py::arg("interleaved") = false, py::arg("index") = none,
          py::arg("status") = none, py::arg("places") = none);
    m.def("paged_free", &paged_free, py::arg("page_table"), py::arg("lengths"), py::arg("refs"), py::arg("slots"),
          py::arg("page_size"), py::arg("status") = none);
    m.def("paged_reserve", &paged_reserve, py::arg("page_table"), py::arg("lengths"), py::arg("refs"), py::arg("slots"),
          py::arg("new_lengths"), py::arg("page_size"), py::arg("status") = none);
    m.def("paged_fork", &paged_fork, py::arg("k_pages"), py::arg("v_pages"), py::arg("page_table"), py::arg("lengths"),
          py::arg("refs"), py::arg("parents"), py::arg("children"), py::arg("status") = none);
    m.def("paged_accept", &paged_accept, py::arg("k_pages"), py::arg("v_pages"), py::arg("page_table"), py::arg("lengths"),
          py::arg("refs"), py::arg("slots"), py::arg("parents"), py::arg("tokens"), py::arg("chosen"),
          py::arg("q_starts") = none, py::arg("index") = none, py::arg("status") = none);
    m.def("paged_copy", &paged_copy, py::arg("k_pages"), py::arg("v_pages"), py::arg("src"), py::arg("dst"),
          py::arg("dst_k_pages") = none, py::arg("dst_v_pages") = none, py::arg("index") = none,
          py::arg("dst_index") = none, py::arg("status") = none);
    m.def("paged_compact", &paged_compact, py::arg("k_pages"), py::arg("v_pages"), py::arg("page_table"),
          py::arg("refs"), py::arg("out_k_pages"), py::arg("out_v_pages"), py::arg("out_table"), py::arg("out_refs"),
          py::arg("index") = none, py::arg("out_index") = none, py::arg("status") = none);
    m.def("paged_attend", &attend, py::arg("q"), py::arg("k_pages"), py::arg("v_pages"), py::arg("page_table"),
          py::arg("lengths"), py::arg("slots"), py::arg("layer"), py::arg("q_starts") = none,
          py::arg("group_starts") = none, py::arg("prefix_pages") = none, py::arg("scale") = none,
          py::arg("status") = none);
    m.def("paged_window_attend", &window_attend, py::arg("q"), py::arg("k_pages"), py::arg("v_pages"),
          py::arg("page_table"), py::arg("lengths"), py::arg("slots"), py::arg("layer"), py::arg("window"),
          py::arg("sinks") = 0, py::arg("q_starts") = none, py::arg("scale") = none, py::arg("status") = none);
    m.def("paged_tree_attend", &tree_attend, py::arg("q"), py::arg("k_pages"), py::arg("v_pages"), py::arg("page_table"),
          py::arg("lengths"), py::arg("slots"), py::arg("parents"), py::arg("layer"), py::arg("q_starts") = none,
          py::arg("scale") = none, py::arg("status") = none);
    m.def("paged_sparse_attend", &sparse_attend, py::arg("q"), py::arg("k_pages"), py::arg("v_pages"), py::arg("index"),
          py::arg("page_table"), py::arg("slots"), py::arg("positions"), py::arg("layer"), py::arg("top_k"),
          py::arg("scale") = none, py::arg("status") = none);
}
