// Host side of the paged cache's operators: argument checks, allocations and the C-ABI calls.  They serve, so there are no autograd nodes.
#include "dsa_host.h"

namespace {

// The tensor itself where its rows can be read 16 bytes at a time in place, a contiguous copy otherwise
Tensor rows_in_place(const Tensor &x) {
    const bool ok = x.numel() == 0 || (x.stride(2) == 1 && (x.size(1) == 1 || x.stride(1) % 8 == 0) && (x.size(0) == 1 || x.stride(0) % 8 == 0) && aligned16(x));
    if (ok) return x;
    const Tensor c = x.contiguous();
    return aligned16(c) ? c : c.clone();
}
// int64 numbers that no int32 holds as the nearest that one does: nowhere, beyond every table
Tensor as_int(const Tensor &x, const char *name) {
    TORCH_CHECK_VALUE(x.scalar_type() == at::kInt || x.scalar_type() == at::kLong, name, " must be int32 or int64, not ", x.scalar_type());
    return x.scalar_type() == at::kInt ? x : x.clamp(INT32_MIN, INT32_MAX).to(at::kInt);
}

struct Cache {
    Tensor table, cu;
    dsa_cache_args args;
    int64_t N;
};
// every tensor of a call lies on the device of `like`
Cache cache_of(const Tensor &like, const Tensor &k, const Tensor &v, const OptTensor &k_scale, const OptTensor &v_scale, const Tensor &table_, const Tensor &cu_) {
    const Tensor none;
    const Tensor &ks = k_scale ? *k_scale : none, &vs = v_scale ? *v_scale : none;
    for (const Tensor *t : {&like, &k, &v, &ks, &vs, &table_, &cu_}) {
        need_gpu(*t);
        if (t->defined()) same_device(like, *t, "a tensor");
    }
    TORCH_CHECK_VALUE(k.dim() == 4 && (k.scalar_type() == at::kBFloat16 || k.scalar_type() == at::kFloat8_e4m3fn), "the cache's keys must be (pages, heads, page, head_dim) bf16 or float8_e4m3fn");
    TORCH_CHECK_VALUE(v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type(), "the cache's values must be like its keys: ", v.sizes(), " ", v.scalar_type(), ", not ", k.sizes(), " ",
                      k.scalar_type());
    const bool e4m3 = k.scalar_type() == at::kFloat8_e4m3fn;
    const int64_t pages = k.size(0), heads = k.size(1), page = k.size(2), dim = k.size(3);
    TORCH_CHECK_VALUE(pages <= INT32_MAX && heads <= INT32_MAX && page <= 256 && dim <= 256, "a cache of ", k.sizes(), ": pages hold up to 256 rows of up to 256");
    auto inside = [&](const Tensor &t, int64_t row) {     // a page's rows are contiguous
        return t.numel() == 0 || ((row == 1 || t.stride(3) == 1) && (page == 1 || t.stride(2) == row) && (heads == 1 || t.stride(1) == page * row) &&
                                  (pages == 1 || t.stride(0) >= heads * page * row) && aligned16(t));
    };
    TORCH_CHECK_VALUE(inside(k, dim) && inside(v, dim), "a page's rows must be contiguous, on a 16-byte boundary and apart from other pages'");
    TORCH_CHECK_VALUE(ks.defined() == e4m3 && vs.defined() == e4m3, "a cache of e4m3 values has scales, one of bf16 values has none");
    if (e4m3)
        for (const Tensor *t : {&ks, &vs}) {
            TORCH_CHECK_VALUE(t->dim() == 3 && t->size(0) == pages && t->size(1) == heads && t->size(2) == page &&
                                  (t->scalar_type() == at::kFloat8_e8m0fnu || t->scalar_type() == at::kByte),
                              "scales must be (", pages, ", ", heads, ", ", page, ") float8_e8m0fnu (or its bytes)");
            TORCH_CHECK_VALUE(inside(*t, 1), "a page's scales must be contiguous, on a 16-byte boundary and apart from other pages'");
        }
    Cache c;
    c.cu = checked_cu(cu_);
    c.N = c.cu.numel() - 1;
    TORCH_CHECK_VALUE(table_.dim() == 2 && table_.size(0) == c.N && table_.size(1) <= INT32_MAX, "page_table must be (", c.N, ", pages of the longest request), not ", table_.sizes());
    c.table = as_int(table_, "page_table");
    if (!(c.table.numel() == 0 || ((c.table.size(1) == 1 || c.table.stride(1) == 1) && (c.N == 1 || c.table.stride(0) >= c.table.size(1))))) c.table = c.table.contiguous();
    auto to_next = [&](const Tensor &t, int64_t row) { return pages > 1 ? t.stride(0) : heads * page * row; };
    c.args = dsa_cache_args{ptr(k), ptr(v), ptr(ks), ptr(vs), to_next(k, dim), to_next(v, dim), e4m3 ? to_next(ks, 1) : 0, e4m3 ? to_next(vs, 1) : 0, iptr(c.table),
                            c.N > 1 ? c.table.stride(0) : c.table.size(1), (int)pages, (int)page, (int)c.table.size(1), (int)heads, (int)dim,
                            e4m3 ? DSA_CACHE_E4M3 : DSA_CACHE_BF16};
    return c;
}
Tensor per_request(const Tensor &x, const Tensor &like, int64_t N, const char *name) {
    need_gpu(x);
    same_device(like, x, name);
    TORCH_CHECK_VALUE(x.dim() == 1 && x.size(0) == N, name, " must hold one number for each of ", N, " requests, not ", x.sizes());
    return as_int(x, name).contiguous();
}

void kv_cache_write(const Tensor &k_pages, const Tensor &v_pages, const OptTensor &k_scale, const OptTensor &v_scale, const Tensor &k_, const Tensor &v_, const Tensor &table,
                    const Tensor &cu, const Tensor &lengths_) {
    const Tensor none;
    no_forward_mode({&k_pages, &v_pages, &k_, &v_}, "kv_cache_write");
    no_graph({&k_pages, &v_pages, &k_, &v_}, "kv_cache_write");
    need_gpu(k_);
    const c10::OptionalDeviceGuard guard(k_.device());
    at::AutoDispatchBelowADInplaceOrView below;
    const Cache c = cache_of(k_, k_pages, v_pages, k_scale, v_scale, table, cu);
    for (const Tensor *t : {&k_, &v_}) {
        same_device(k_, *t, "v");
        check_bf16_thd(*t, t == &k_ ? "k" : "v");
        TORCH_CHECK_VALUE(t->size(0) == k_.size(0) && t->size(1) == c.args.Hkv && t->size(2) == c.args.D, "k and v must be (T, ", c.args.Hkv, ", ", c.args.D, "), not ", t->sizes());
    }
    TORCH_CHECK_VALUE(k_.size(0) <= INT32_MAX, "too many rows: ", k_.size(0));
    const Tensor lengths = per_request(lengths_, k_, c.N, "lengths"), k = rows_in_place(k_), v = rows_in_place(v_);
    check(dsa_cache_write(&c.args, ptr(k), tok_of(k), head_of(k), ptr(v), tok_of(v), head_of(v), iptr(c.cu), iptr(lengths), (int)k.size(0), (int)c.N, stream_of(k)), "dsa_cache_write");
    for (const Tensor *t : {&k_pages, &v_pages, k_scale ? &*k_scale : &none, v_scale ? &*v_scale : &none})
        if (t->defined() && !t->is_inference()) torch::autograd::impl::bump_version(*t);
}

std::vector<Tensor> kv_cache_read(const Tensor &k_pages, const Tensor &v_pages, const OptTensor &k_scale, const OptTensor &v_scale, const Tensor &table, const Tensor &cu,
                                  int64_t rows, const OptTensor &first_) {
    no_forward_mode({&k_pages, &v_pages}, "kv_cache_read");
    no_graph({&k_pages, &v_pages}, "kv_cache_read");
    need_gpu(k_pages);
    const c10::OptionalDeviceGuard guard(k_pages.device());
    at::AutoDispatchBelowADInplaceOrView below;
    const Cache c = cache_of(k_pages, k_pages, v_pages, k_scale, v_scale, table, cu);
    TORCH_CHECK_VALUE(rows >= 0 && rows <= INT32_MAX, "rows must be a number of rows, not ", rows);
    const Tensor first = first_ ? per_request(*first_, k_pages, c.N, "first") : Tensor();
    const Tensor k = empty({rows, c.args.Hkv, c.args.D}, at::kBFloat16, k_pages), v = empty({rows, c.args.Hkv, c.args.D}, at::kBFloat16, k_pages);
    check(dsa_cache_read(&c.args, iptr(c.cu), iptr(first), (int)rows, (int)c.N, ptr(k), ptr(v), stream_of(k)), "dsa_cache_read");
    return {k, v};
}

std::vector<Tensor> paged_attn(const Tensor &q_, const Tensor &k_pages, const Tensor &v_pages, const OptTensor &k_scale, const OptTensor &v_scale, const Tensor &table, const Tensor &cu,
                               const Tensor &lengths_, std::optional<int64_t> max_new, std::optional<int64_t> max_length, std::optional<double> scale, bool return_lse) {
    no_forward_mode({&q_, &k_pages, &v_pages}, "paged_attn");
    no_graph({&q_, &k_pages, &v_pages}, "paged_attn");
    need_gpu(q_);
    const c10::OptionalDeviceGuard guard(q_.device());
    at::AutoDispatchBelowADInplaceOrView below;
    const Cache c = cache_of(q_, k_pages, v_pages, k_scale, v_scale, table, cu);
    check_bf16_thd(q_, "q");
    const int64_t T = q_.size(0), Hq = q_.size(1), D = q_.size(2);
    TORCH_CHECK_VALUE(D == c.args.D && Hq >= 1 && c.args.Hkv >= 1 && Hq % c.args.Hkv == 0, "q is (T, ", Hq, ", ", D, "), the cache has ", c.args.Hkv, " heads of ", c.args.D);
    TORCH_CHECK_VALUE(T <= INT32_MAX, "too many rows: ", T);
    TORCH_CHECK_VALUE(!max_new || *max_new >= 1, "max_new must be at least 1");
    TORCH_CHECK_VALUE(!max_length || *max_length >= 1, "max_length must be at least 1");
    const int most_new = max_new ? (int)std::min<int64_t>(*max_new, INT32_MAX) : 0, longest = max_length ? (int)std::min<int64_t>(*max_length, INT32_MAX) : 0;
    const Tensor lengths = per_request(lengths_, q_, c.N, "lengths"), q = rows_in_place(q_);
    const Tensor out = empty({T, Hq, D}, at::kBFloat16, q), lse = return_lse ? empty({Hq, T}, at::kFloat, q) : Tensor();
    const size_t bytes = dsa_paged_attn_workspace_bytes(&c.args, (int)T, (int)c.N, (int)Hq, most_new, longest);
    const Tensor ws = bytes ? empty_bytes(bytes, q) : Tensor();
    check(dsa_paged_attn(&c.args, ptr(q), tok_of(q), head_of(q), iptr(c.cu), iptr(lengths), (int)T, (int)c.N, (int)Hq, (float)(scale ? *scale : std::pow((double)D, -0.5)), most_new,
                         longest, ptr(out), fptr(lse), ptr(ws), bytes, stream_of(q)), "dsa_paged_attn");
    return return_lse ? std::vector<Tensor>{out, lse} : std::vector<Tensor>{out};
}

}  // namespace

void bind_cache(py::module_ &m) {
    const auto nogil = py::call_guard<py::gil_scoped_release>();
    m.def("kv_cache_write", &kv_cache_write, nogil);
    m.def("kv_cache_read", &kv_cache_read, nogil);
    m.def("paged_attn", &paged_attn, nogil);
}
