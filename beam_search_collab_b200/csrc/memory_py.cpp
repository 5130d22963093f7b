// memory_py.cpp -- Python binding of the token-memory entries
// (include/bsearch.h) for PyTorch tensors: shapes and types are checked here
// (ValueError), outputs and workspaces come from PyTorch's allocator, and one
// C call does the rest (its failures raise the package's BSearchError).
// Native because a call's kernels take a few microseconds when it is small,
// and the same checks in Python took 20 to 35.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <optional>
#include <string>

#include "bsearch.h"

namespace py = pybind11;
using at::Tensor;
using MaybeTensor = std::optional<Tensor>;

namespace {

PyObject* g_error = nullptr;      // the package's exception class: (status, message)

void need(bool ok, const char* what) {
    if (!ok) throw py::value_error(what);
}

void check(bs_status s) {
    if (s == BS_OK) return;
    py::object e = py::reinterpret_borrow<py::object>(g_error)(static_cast<int>(s), std::string(bs_last_error()));
    PyErr_SetObject(g_error, e.ptr());
    throw py::error_already_set();
}

// A dimension as the C entries take it: one that 32 bits do not hold must not
// become another.
int32_t count(int64_t n) {
    need(n < (int64_t{1} << 31), "a dimension of 2^31 or more is not supported");
    return static_cast<int32_t>(n);
}

int type_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return BS_F32;
        case at::kHalf: return BS_F16;
        case at::kBFloat16: return BS_BF16;
        default: return -1;
    }
}

bool is_type16(const Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }

const int32_t* indexes(const Tensor& t, at::IntArrayRef shape, const char* name, at::Device device) {
    if (t.scalar_type() != at::kInt || !t.is_contiguous() || t.device() != device || t.sizes() != shape)
        throw py::value_error(std::string(name) + " must be a contiguous int32 tensor of the documented shape, on the device of the others");
    return t.const_data_ptr<int32_t>();
}

// [tokens, heads, dim], last dimension contiguous.
void check_rows(const Tensor& t, const char* name, const Tensor* like) {
    if (!t.is_cuda() || t.dim() != 3 || (t.size(2) > 1 && t.stride(2) != 1))
        throw py::value_error(std::string(name) + " must be a CUDA tensor [tokens, heads, dim], last dimension contiguous");
    if (!is_type16(t)) throw py::value_error(std::string(name) + " must be float16 or bfloat16");
    if (like && (t.scalar_type() != like->scalar_type() || t.device() != like->device() || t.size(2) != like->size(2)))
        throw py::value_error(std::string(name) + " must have the type, device and last dimension of the others");
}

// Strides of all dimensions but the last; one that only meets index 0 is 0.
template <size_t N>
void strides(const Tensor& t, int64_t (&out)[N]) {
    for (size_t i = 0; i < N; ++i) out[i] = t.size(i) > 1 ? t.stride(i) : 0;
}

// The stream a call goes to, made PyTorch's current one for as long as the
// call lasts: memory that it asks for is then free on that stream, where its
// kernels run.  Where the caller's current stream is another, PyTorch is told
// who else uses what.
struct Target {
    c10::cuda::CUDAGuard device;
    c10::cuda::CUDAStream callers;
    cudaStream_t stream;
    c10::cuda::OptionalCUDAStreamGuard guard;
    Target(at::Device on, std::optional<uint64_t> handle)
        : device(on), callers(c10::cuda::getCurrentCUDAStream(on.index())), stream(callers.stream()) {
        if (!handle || reinterpret_cast<cudaStream_t>(*handle) == stream) return;
        stream = reinterpret_cast<cudaStream_t>(*handle);
        guard.reset_stream(stream ? c10::cuda::getStreamFromExternal(stream, on.index()) : c10::cuda::getDefaultCUDAStream(on.index()));
    }
    // Tensors of the caller that the kernels use: freed, they are not given
    // out again before the kernels are done.
    void uses(std::initializer_list<const Tensor*> given) const { record(given, c10::cuda::getCurrentCUDAStream(callers.device_index())); }
    // Tensors made here that the caller's stream will use.
    void gives(std::initializer_list<const Tensor*> made) const { record(made, callers); }

private:
    void record(std::initializer_list<const Tensor*> tensors, c10::cuda::CUDAStream other) const {
        if (stream == callers.stream()) return;
        for (const Tensor* t : tensors)
            if (t->defined()) t->record_stream(other);
    }
};

Tensor scratch(size_t bytes, at::Device device) {
    return bytes ? at::empty({static_cast<int64_t>(bytes)}, at::TensorOptions().dtype(at::kByte).device(device)) : Tensor();
}

// These operators have no gradients.  An output made from something that needs
// one says so when a backward pass reaches it, where it would be left out of
// the pass without a word.
struct NoGradient : torch::autograd::Function<NoGradient> {
    static Tensor forward(torch::autograd::AutogradContext*, const Tensor& made, const Tensor&) { return made; }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext*, torch::autograd::variable_list) {
        TORCH_CHECK(false, "the token-memory operators have no gradient: use them under torch.no_grad() or on detached tensors");
        return {};
    }
};

Tensor from(const Tensor& made, std::initializer_list<const Tensor*> inputs) {
    if (made.defined() && at::GradMode::is_enabled())
        for (const Tensor* t : inputs)
            if (t->requires_grad()) return NoGradient::apply(made, *t);
    return made;
}

py::object maybe(const Tensor& t) { return t.defined() ? py::cast(t) : py::none(); }

py::tuple prompt_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu_q, const MaybeTensor& given_cu_k,
                           bool causal, std::optional<double> scale, bool with_lse, std::optional<uint64_t> stream) {
    check_rows(q, "q", nullptr);
    check_rows(k, "k", &q);
    check_rows(v, "v", &q);
    need(k.sizes() == v.sizes(), "k and v must have the same shape");
    need(given_cu_k || q.size(0) == k.size(0), "cu_k is needed when q and k have different numbers of rows");
    const Tensor& cu_k = given_cu_k ? *given_cu_k : cu_q;
    need(cu_q.dim() == 1 && cu_q.size(0) >= 1, "cu_q must be [sequences + 1]");
    bs_prompt_attention_desc d{};
    d.cu_q = indexes(cu_q, {cu_q.size(0)}, "cu_q", q.device());
    d.cu_k = indexes(cu_k, {cu_q.size(0)}, "cu_k", q.device());
    Target to(q.device(), stream);
    const Tensor out = at::empty(q.sizes(), q.options());
    const Tensor lse = with_lse ? at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat)) : Tensor();
    d.q = q.const_data_ptr();
    d.k = k.const_data_ptr();
    d.v = v.const_data_ptr();
    d.out = out.data_ptr();
    d.lse = with_lse ? lse.data_ptr<float>() : nullptr;
    strides(q, d.q_stride);
    strides(k, d.k_stride);
    strides(v, d.v_stride);
    d.total_q = count(q.size(0));
    d.total_k = count(k.size(0));
    d.num_seqs = count(cu_q.size(0) - 1);
    d.q_heads = count(q.size(1));
    d.kv_heads = count(k.size(1));
    d.dim = count(q.size(2));
    d.dtype = type_of(q);
    d.causal = causal;
    d.scale = static_cast<float>(scale ? *scale : 1.0 / std::sqrt(static_cast<double>(std::max<int64_t>(q.size(2), 1))));
    size_t bytes = 0;
    check(bs_prompt_attention_workspace(&d, &bytes));
    const Tensor work = scratch(bytes, q.device());
    d.workspace = bytes ? work.data_ptr() : nullptr;
    d.workspace_bytes = bytes;
    check(bs_prompt_attention(&d, to.stream));
    to.uses({&q, &k, &v, &cu_q, &cu_k});
    to.gives({&out, &lse});
    return py::make_tuple(from(out, {&q, &k, &v}), maybe(from(lse, {&q, &k})));
}

struct Cache {
    Tensor k, v, k_scale, v_scale;
    bs_token_cache c{};

    Cache(const Tensor& k_, const Tensor& v_, const Tensor& ks, const Tensor& vs) : k(k_), v(v_), k_scale(ks), v_scale(vs) {
        need(k.is_cuda() && k.dim() == 4 && k.scalar_type() == at::kChar && k.is_contiguous(),
             "k must be a contiguous CUDA int8 tensor [blocks, kv_heads, block, dim]");
        need(v.sizes() == k.sizes() && v.scalar_type() == at::kChar && v.device() == k.device() && v.is_contiguous(), "v must be like k");
        for (const Tensor* s : {&k_scale, &v_scale})
            need(s->dim() == 2 && s->size(0) == k.size(0) && s->size(1) == k.size(1) && s->scalar_type() == at::kFloat &&
                     s->device() == k.device() && s->is_contiguous(),
                 "scales must be contiguous float32 tensors [blocks, kv_heads]");
        c.k = static_cast<int8_t*>(k.data_ptr());
        c.v = static_cast<int8_t*>(v.data_ptr());
        c.k_scale = k_scale.data_ptr<float>();
        c.v_scale = v_scale.data_ptr<float>();
        c.num_blocks = count(k.size(0));
        c.kv_heads = count(k.size(1));
        c.block = count(k.size(2));
        c.dim = count(k.size(3));
    }

    void write(const Tensor& x, const Tensor& y, const Tensor& cu, const Tensor& table, const Tensor& start,
               std::optional<uint64_t> stream) const {
        check_rows(x, "k", nullptr);
        check_rows(y, "v", &x);
        need(x.sizes() == y.sizes() && x.size(1) == k.size(1) && x.size(2) == k.size(3) && x.device() == k.device(),
             "k and v must be [tokens, kv_heads, dim] of the cache, on its device");
        need(table.dim() == 2, "table must be [sequences, width]");
        const int64_t n = table.size(0);
        bs_cache_write_desc d{};
        d.cu = indexes(cu, {n + 1}, "cu", k.device());
        d.table = indexes(table, table.sizes(), "table", k.device());
        d.start = indexes(start, {n}, "start", k.device());
        Target to(k.device(), stream);
        d.k = x.const_data_ptr();
        d.v = y.const_data_ptr();
        strides(x, d.k_stride);
        strides(y, d.v_stride);
        d.total = count(x.size(0));
        d.num_seqs = count(n);
        d.table_width = count(table.size(1));
        d.dtype = type_of(x);
        check(bs_cache_write(&c, &d, to.stream));
        to.uses({&k, &v, &k_scale, &v_scale, &x, &y, &cu, &table, &start});
    }

    py::tuple read(const Tensor& table, const Tensor& lens, const Tensor& positions, at::ScalarType dtype, bool keys, bool values,
                   std::optional<uint64_t> stream) const {
        need(dtype == at::kFloat || dtype == at::kHalf || dtype == at::kBFloat16, "dtype must be float32, float16 or bfloat16");
        need(table.dim() == 2, "table must be [sequences, width]");
        const int64_t n = table.size(0), heads = k.size(1);
        need(positions.scalar_type() == at::kInt && positions.device() == k.device() && (positions.dim() == 2 || positions.dim() == 3) &&
                 positions.size(0) == n && (positions.dim() == 2 || positions.size(1) == heads) &&
                 (positions.size(-1) <= 1 || positions.stride(-1) == 1),
             "positions must be int32 [sequences, n] or [sequences, kv_heads, n], last dimension contiguous");
        bs_cache_read_desc d{};
        d.table = indexes(table, table.sizes(), "table", k.device());
        d.lens = indexes(lens, {n}, "lens", k.device());
        d.positions = positions.const_data_ptr<int32_t>();
        d.position_seq_stride = n > 1 ? positions.stride(0) : 0;
        d.position_head_stride = positions.dim() == 3 && heads > 1 ? positions.stride(1) : 0;
        Target to(k.device(), stream);
        const at::TensorOptions options = at::TensorOptions().dtype(dtype).device(k.device());
        const Tensor a = keys ? at::empty({n, heads, positions.size(-1), k.size(3)}, options) : Tensor();
        const Tensor b = values ? at::empty({n, heads, positions.size(-1), k.size(3)}, options) : Tensor();
        d.k = keys ? a.data_ptr() : nullptr;
        d.v = values ? b.data_ptr() : nullptr;
        d.num_seqs = count(n);
        d.table_width = count(table.size(1));
        d.count = count(positions.size(-1));
        d.dtype = dtype == at::kFloat ? BS_F32 : dtype == at::kHalf ? BS_F16 : BS_BF16;
        check(bs_cache_read(&c, &d, to.stream));
        to.uses({&k, &v, &k_scale, &v_scale, &table, &lens, &positions});
        to.gives({&a, &b});
        return py::make_tuple(maybe(a), maybe(b));
    }

    py::tuple attention(const Tensor& q, const Tensor& table, const Tensor& lens, std::optional<double> scale, bool with_lse,
                        const MaybeTensor& mass, bool with_mass, const MaybeTensor& given_out, std::optional<uint64_t> stream) const {
        need(q.dim() == 4 && q.device() == k.device() && is_type16(q) && q.size(3) == k.size(3) && (q.size(3) <= 1 || q.stride(3) == 1),
             "q must be float16 or bfloat16 [sequences, queries, q_heads, dim] on the cache's device, last dimension contiguous");
        need(table.dim() == 2 && table.size(0) == q.size(0), "table must be [sequences, width], q have as many sequences");
        const int64_t n = table.size(0), heads = k.size(1);
        bs_cache_attention_desc d{};
        d.table = indexes(table, table.sizes(), "table", k.device());
        d.lens = indexes(lens, {n}, "lens", k.device());
        Target to(k.device(), stream);
        const Tensor out = at::empty(q.sizes(), q.options());
        const Tensor lse = with_lse ? at::empty({n, q.size(1), q.size(2)}, q.options().dtype(at::kFloat)) : Tensor();
        Tensor sum;
        if (given_out) sum = *given_out;
        else if (mass) sum = at::empty(mass->sizes(), mass->options());
        else if (with_mass) sum = at::empty({n, heads, table.size(1) * k.size(2)}, q.options().dtype(at::kFloat));
        if (sum.defined()) {
            for (const Tensor* m : {mass ? &*mass : &sum, static_cast<const Tensor*>(&sum)})
                need(m->scalar_type() == at::kFloat && m->device() == k.device() && m->dim() == 3 && m->is_contiguous() &&
                         m->sizes() == sum.sizes() && m->size(0) == n && m->size(1) == heads,
                     "mass must be contiguous float32 [sequences, kv_heads, width]");
            d.mass = mass ? mass->const_data_ptr<float>() : nullptr;
            d.out_mass = sum.data_ptr<float>();
            d.mass_width = count(sum.size(2));
        }
        d.q = q.const_data_ptr();
        strides(q, d.q_stride);
        d.out = out.data_ptr();
        d.lse = with_lse ? lse.data_ptr<float>() : nullptr;
        d.num_seqs = count(n);
        d.table_width = count(table.size(1));
        d.queries = count(q.size(1));
        d.q_heads = count(q.size(2));
        d.dtype = type_of(q);
        d.scale = static_cast<float>(scale ? *scale : 1.0 / std::sqrt(static_cast<double>(std::max<int64_t>(q.size(3), 1))));
        size_t bytes = 0;
        check(bs_cache_attention_workspace(&c, &d, &bytes));
        const Tensor work = scratch(bytes, k.device());
        d.workspace = bytes ? work.data_ptr() : nullptr;
        d.workspace_bytes = bytes;
        check(bs_cache_attention(&c, &d, to.stream));
        to.uses({&k, &v, &k_scale, &v_scale, &q, &table, &lens});
        if (mass) to.uses({&*mass});
        if (given_out) to.uses({&sum});
        else to.gives({&sum});
        to.gives({&out, &lse});
        if (!given_out) sum = mass ? from(sum, {&q, &*mass}) : from(sum, {&q});
        return py::make_tuple(from(out, {&q}), maybe(from(lse, {&q})), maybe(sum));
    }

    py::tuple evict(const Tensor& mass, const Tensor& table, const Tensor& lens, const Tensor& new_table, int64_t budget, int64_t sinks,
                    int64_t recent, std::optional<uint64_t> stream) const {
        need(table.dim() == 2 && new_table.dim() == 2, "table and new_table must be [sequences, width]");
        const int64_t n = table.size(0), heads = k.size(1);
        need(mass.scalar_type() == at::kFloat && mass.device() == k.device() && mass.is_contiguous() && mass.dim() == 3 &&
                 mass.size(0) == n && mass.size(1) == heads,
             "mass must be contiguous float32 [sequences, kv_heads, width]");
        need(budget > 0 && budget < (1 << 30), "budget must be positive and below 2^30");
        need(sinks >= 0 && recent >= 0 && sinks <= budget && recent <= budget, "sinks and recent must be in 0 .. budget");
        bs_cache_evict_desc d{};
        d.mass = mass.const_data_ptr<float>();
        d.table = indexes(table, table.sizes(), "table", k.device());
        d.lens = indexes(lens, {n}, "lens", k.device());
        d.new_table = indexes(new_table, {n, new_table.size(1)}, "new_table", k.device());
        Target to(k.device(), stream);
        const at::TensorOptions ints = lens.options();
        const Tensor kept = at::empty({n, heads, budget}, ints), new_lens = at::empty({n}, ints);
        const Tensor new_mass = at::empty({n, heads, budget}, mass.options());
        d.kept = kept.data_ptr<int32_t>();
        d.new_lens = new_lens.data_ptr<int32_t>();
        d.new_mass = new_mass.data_ptr<float>();
        d.num_seqs = count(n);
        d.table_width = count(table.size(1));
        d.new_table_width = count(new_table.size(1));
        d.mass_width = count(mass.size(2));
        d.budget = budget;
        d.sinks = sinks;
        d.recent = recent;
        size_t bytes = 0;
        check(bs_cache_evict_workspace(&c, &d, &bytes));
        const Tensor work = scratch(bytes, k.device());
        d.workspace = bytes ? work.data_ptr() : nullptr;
        d.workspace_bytes = bytes;
        check(bs_cache_evict(&c, &d, to.stream));
        to.uses({&k, &v, &k_scale, &v_scale, &mass, &table, &lens, &new_table});
        to.gives({&kept, &new_lens, &new_mass});
        return py::make_tuple(kept, new_lens, from(new_mass, {&mass}));
    }
};

uint32_t take_errors(int64_t device, std::optional<uint64_t> stream) {
    Target to(at::Device(at::kCUDA, static_cast<c10::DeviceIndex>(device)), stream);
    uint32_t flags = 0;
    bs_status s;
    {
        py::gil_scoped_release others;       // it waits for the stream
        s = bs_memory_take_errors(to.stream, &flags);
    }
    check(s);
    return flags;
}

}  // namespace

PYBIND11_MODULE(_memory, m) {
    m.def("set_error", [](py::object e) { g_error = e.release().ptr(); });
    m.def("prompt_attention", &prompt_attention);
    m.def("take_errors", &take_errors);
    py::class_<Cache>(m, "Cache")
        .def(py::init<const Tensor&, const Tensor&, const Tensor&, const Tensor&>())
        .def_readonly("k", &Cache::k)
        .def_readonly("v", &Cache::v)
        .def_readonly("k_scale", &Cache::k_scale)
        .def_readonly("v_scale", &Cache::v_scale)
        .def("_write", &Cache::write)
        .def("_read", &Cache::read)
        .def("_attention", &Cache::attention)
        .def("_evict", &Cache::evict);
}
