// Row groups and linear maps with the weights of a row's group as torch library ops (see oeq_torch.cpp for why they are native).
//
// The map Z = F(x, w) is linear in rows and in weights, and its gradients T(dz, w) and G(x, dz) are made of the same three
// products: one op with a `kind` is closed under differentiation, so derivatives of any order run these kernels.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/library.h>

#include <map>
#include <mutex>
#include <optional>
#include <string>
#include <string_view>
#include <tuple>
#include <vector>

#include "oeq_torch_common.h"

namespace {

using at::Tensor;
using oeq_torch::check;
using oeq_torch::direct;
using oeq_torch::index_ptr;

enum Kind { PRODUCT = 0, INPUT = 1, WEIGHTS = 2 };      // F(x, w), T(dz, w), G(x, dz)

// A map is named by its irreps, "8x0e+4x1o->6x0e+4x1o": a traced graph that is saved holds the name, and another process makes the map when
// it first meets it.  Maps live as long as the process: an autograd graph may hold one after its front end has gone.
struct Linear {
    std::string name;
    oeq_grouped* handle;
    int64_t in, out, numel;
    int64_t width(int64_t kind) const { return kind == PRODUCT ? out : (kind == INPUT ? in : numel); }     // of a result
    int64_t width_a(int64_t kind) const { return kind == INPUT ? out : in; }
    int64_t width_b(int64_t kind) const { return kind == WEIGHTS ? out : numel; }
};
// "8x0e+4x1o" -> its blocks and their width; false if it is anything else.
bool read_irreps(std::string_view s, std::vector<oeq_irrep>& blocks, int64_t& dim) {
    dim = 0;
    auto number = [&](int32_t& v) {
        size_t n = 0;
        for (v = 0; n < s.size() && n < 9 && s[n] >= '0' && s[n] <= '9'; ++n) v = 10 * v + (s[n] - '0');
        s.remove_prefix(n);
        return n > 0;
    };
    auto one_of = [&](std::string_view chars) {
        const char c = !s.empty() && chars.find(s[0]) != chars.npos ? s[0] : '\0';
        if (c) s.remove_prefix(1);
        return c;
    };
    while (!s.empty()) {
        oeq_irrep b{};
        if (!number(b.mul) || !one_of("x") || !number(b.l)) return false;
        const char parity = one_of("eo");
        if (!parity) return false;
        b.parity = parity == 'e' ? 1 : -1;
        blocks.push_back(b);
        dim += (int64_t)b.mul * (2 * b.l + 1);
        if (!s.empty() && (!one_of("+") || s.empty())) return false;
    }
    return true;
}
std::mutex linear_mutex;
// Makes the map if it is not known yet: an OEQ code (oeq_last_error has the reason).
int find_linear(std::string_view name, const Linear*& found) {
    static auto* known = new std::map<std::string, Linear, std::less<>>();      // (elements of a map stay where they are)
    std::lock_guard<std::mutex> lock(linear_mutex);
    auto at = known->find(name);
    if (at == known->end()) {
        const size_t arrow = name.find("->");
        std::vector<oeq_irrep> in, out;
        Linear lin{std::string(name), nullptr, 0, 0, 0};
        TORCH_CHECK_VALUE(arrow != name.npos && read_irreps(name.substr(0, arrow), in, lin.in) && read_irreps(name.substr(arrow + 2), out, lin.out),
                          "a linear map is named by its irreps, as in 8x0e+4x1o->6x0e, got ", name);
        if (int rc = oeq_grouped_create(in.data(), (int)in.size(), out.data(), (int)out.size(), &lin.handle)) return rc;
        lin.numel = oeq_grouped_weight_numel(lin.handle);
        at = known->emplace(lin.name, lin).first;
    }
    found = &at->second;
    return OEQ_OK;
}
const Linear& linear_of(std::string_view name, int64_t kind) {
    TORCH_CHECK_VALUE(kind >= PRODUCT && kind <= WEIGHTS, "no such product of a linear map: ", kind);
    const Linear* lin = nullptr;
    check(find_linear(name, lin));
    return *lin;
}

int dtype_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return OEQ_F32;
        case at::kDouble: return OEQ_F64;
        case at::kBFloat16: return OEQ_BF16;
        case at::kHalf: return OEQ_F16;
        default: TORCH_CHECK_VALUE(false, "tensors must be float32, float64, bfloat16 or float16, got ", t);
    }
}

void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

// ---------------------------------------------------------------- row groups
void check_groups(int64_t rows, int64_t groups) {
    TORCH_CHECK_VALUE(groups >= 1 && groups <= OEQ_MOST_GROUPS, "the number of groups must be in 1 .. ", OEQ_MOST_GROUPS, ", got ", groups);
    TORCH_CHECK_VALUE(rows >= 0 && rows < (int64_t(1) << 31), "the number of rows must be in 0 .. 2^31 - 1, got ", rows);
}
std::tuple<Tensor, Tensor, Tensor, Tensor> row_groups_cuda(const Tensor& index_in, int64_t groups) {
    TORCH_CHECK_VALUE(index_in.dim() == 1 && index_in.scalar_type() == at::kLong, "the groups of the rows must be a 1-D int64 tensor, got ",
                      index_in.sizes(), " of ", index_in.scalar_type());
    const int64_t rows = index_in.size(0);
    check_groups(rows, groups);
    const auto index = index_in.expect_contiguous();
    c10::cuda::CUDAGuard guard(index->device());
    Tensor order = at::empty_like(*index), slots = at::empty_like(*index), offsets = at::empty({groups + 1}, index->options());
    Tensor blocks = at::empty({oeq_row_groups_blocks(rows, groups), 3}, index->options().dtype(at::kInt));
    const size_t bytes = oeq_row_groups_workspace_bytes(rows, groups);
    Tensor ws;
    if (bytes) ws = at::empty({(int64_t)bytes}, index->options().dtype(at::kByte));
    check(oeq_row_groups(rows, groups, index_ptr(*index), order.mutable_data_ptr<int64_t>(), slots.mutable_data_ptr<int64_t>(),
                         offsets.mutable_data_ptr<int64_t>(), blocks.mutable_data_ptr<int32_t>(), bytes ? ws.mutable_data_ptr() : nullptr, bytes, stream()));
    return {order, slots, offsets, blocks};
}
std::tuple<Tensor, Tensor, Tensor> row_groups_from_counts_cuda(const Tensor& counts_in, int64_t rows) {
    TORCH_CHECK_VALUE(counts_in.dim() == 1 && counts_in.scalar_type() == at::kLong, "the numbers of rows must be a 1-D int64 tensor, got ",
                      counts_in.sizes(), " of ", counts_in.scalar_type());
    const int64_t groups = counts_in.size(0);
    check_groups(rows, groups);
    const auto counts = counts_in.expect_contiguous();
    c10::cuda::CUDAGuard guard(counts->device());
    Tensor index = at::empty({rows}, counts->options()), offsets = at::empty({groups + 1}, counts->options());
    Tensor blocks = at::empty({oeq_row_groups_blocks(rows, groups), 3}, counts->options().dtype(at::kInt));
    check(oeq_row_groups_from_counts(rows, groups, index_ptr(*counts), index.mutable_data_ptr<int64_t>(), offsets.mutable_data_ptr<int64_t>(),
                                     blocks.mutable_data_ptr<int32_t>(), stream()));
    return {index, offsets, blocks};
}

// ---------------------------------------------------------------- the product and its gradients
Tensor run_linear(const Linear& lin, const Tensor& a_in, const Tensor& b_in, const std::optional<Tensor>& order_in, const Tensor& offsets_in,
                  const Tensor& blocks_in, int64_t kind) {
    const int dtype = dtype_of(a_in.scalar_type());
    const char* names[3][2] = {{"rows", "weights"}, {"output gradient", "weights"}, {"rows", "output gradient"}};
    TORCH_CHECK_VALUE(offsets_in.dim() == 1 && offsets_in.size(0) >= 2 && offsets_in.scalar_type() == at::kLong, "offsets must be a 1-D int64 tensor");
    const int64_t groups = offsets_in.size(0) - 1;
    TORCH_CHECK_VALUE(a_in.dim() == 2 && a_in.size(1) == lin.width_a(kind), names[kind][0], " must be [rows, ", lin.width_a(kind), "], got ", a_in.sizes());
    const int64_t rows = a_in.size(0);
    TORCH_CHECK_VALUE(b_in.dim() == 2 && b_in.size(0) == (kind == WEIGHTS ? rows : groups) && b_in.size(1) == lin.width_b(kind), names[kind][1], " must be [",
                      kind == WEIGHTS ? rows : groups, ", ", lin.width_b(kind), "], got ", b_in.sizes());
    TORCH_CHECK_VALUE(a_in.scalar_type() == b_in.scalar_type(), "tensors must be of one type, got ", a_in.scalar_type(), " and ", b_in.scalar_type());
    check_groups(rows, groups);
    TORCH_CHECK_VALUE(!order_in || (order_in->dim() == 1 && order_in->size(0) == rows && order_in->scalar_type() == at::kLong),
                      "the groups are those of another number of rows");
    TORCH_CHECK_VALUE(blocks_in.dim() == 2 && blocks_in.size(1) == 3 && blocks_in.size(0) == oeq_row_groups_blocks(rows, groups) &&
                          blocks_in.scalar_type() == at::kInt, "the groups are those of another number of rows");
    TORCH_CHECK_VALUE(b_in.device() == a_in.device() && offsets_in.device() == a_in.device() && blocks_in.device() == a_in.device() &&
                          (!order_in || order_in->device() == a_in.device()), "tensors must be on one device");
    const auto a = a_in.expect_contiguous(), b = b_in.expect_contiguous(), offsets = offsets_in.expect_contiguous(), blocks = blocks_in.expect_contiguous();
    const Tensor order = order_in ? order_in->contiguous() : Tensor();
    const int64_t* order_ptr = order_in ? index_ptr(order) : nullptr;
    c10::cuda::CUDAGuard guard(a->device());
    const int32_t* table = static_cast<const int32_t*>(blocks->const_data_ptr());
    Tensor out = at::empty({kind == WEIGHTS ? groups : rows, lin.width(kind)}, a->options());
    if (kind == WEIGHTS) {
        const size_t bytes = oeq_grouped_workspace_bytes(lin.handle, dtype, rows, groups);
        Tensor ws;
        if (bytes) ws = at::empty({(int64_t)bytes}, a->options().dtype(at::kByte));
        check(oeq_grouped_backward_weights(lin.handle, dtype, rows, groups, a->const_data_ptr(), b->const_data_ptr(), order_ptr, index_ptr(*offsets),
                                           out.mutable_data_ptr(), bytes ? ws.mutable_data_ptr() : nullptr, bytes, stream()));
    } else {
        auto* call = kind == PRODUCT ? oeq_grouped_forward : oeq_grouped_backward_input;
        check(call(lin.handle, dtype, rows, groups, a->const_data_ptr(), b->const_data_ptr(), order_ptr, index_ptr(*offsets), table, out.mutable_data_ptr(),
                   stream()));
    }
    return out;
}

Tensor linear_cuda(const Tensor& a, const Tensor& b, const std::optional<Tensor>& order, const Tensor& offsets, const Tensor& blocks, std::string_view name,
                   int64_t kind) {
    return run_linear(linear_of(name, kind), a, b, order, offsets, blocks, kind);
}

using Signature = Tensor(const Tensor&, const Tensor&, const std::optional<Tensor>&, const Tensor&, const Tensor&, std::string_view, int64_t);

Tensor call_linear(const Linear& lin, const Tensor& a, const Tensor& b, const std::optional<Tensor>& order, const Tensor& offsets, const Tensor& blocks,
                   int64_t kind) {
    if (direct({a, b, offsets, blocks})) return run_linear(lin, a, b, order, offsets, blocks, kind);
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("openequivariance_b200::grouped_linear", "").typed<Signature>();
    return op.call(a, b, order, offsets, blocks, lin.name, kind);
}

struct LinearNode final : torch::autograd::Node {
    const Linear* lin;
    int64_t kind;
    bool has_order;
    torch::autograd::SavedVariable a, b, order, offsets, blocks;
    std::string name() const override { return "OeqGroupedLinearBackward"; }
    // (saved operands live as long as the graph, as those of the other operators' nodes)
    torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
        if (!grads[0].defined()) return {Tensor(), Tensor()};
        const Tensor& e = grads[0];
        Tensor x, y, off, blk;
        std::optional<Tensor> ord;
        {
            std::lock_guard<std::mutex> lock(mutex_);
            x = a.unpack();
            y = b.unpack();
            off = offsets.unpack();
            blk = blocks.unpack();
            if (has_order) ord = order.unpack();
        }
        auto call = [&](int64_t k, const Tensor& p, const Tensor& q) { return call_linear(*lin, p, q, ord, off, blk, k); };
        Tensor ga, gb;
        if (task_should_compute_output(0)) ga = kind == PRODUCT ? call(INPUT, e, y) : (kind == INPUT ? call(PRODUCT, e, y) : call(INPUT, y, e));
        if (task_should_compute_output(1)) gb = kind == PRODUCT ? call(WEIGHTS, x, e) : (kind == INPUT ? call(WEIGHTS, e, x) : call(PRODUCT, x, e));
        return {ga, gb};
    }
};

Tensor linear_autograd(const Tensor& a, const Tensor& b, const std::optional<Tensor>& order, const Tensor& offsets, const Tensor& blocks,
                       std::string_view name, int64_t kind) {
    TORCH_CHECK_NOT_IMPLEMENTED(!torch::autograd::isFwGradDefined(a) && !torch::autograd::isFwGradDefined(b),
                                "openequivariance_b200: the operators have no forward-mode derivative");
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("openequivariance_b200::grouped_linear", "").typed<Signature>();
    std::shared_ptr<LinearNode> node;
    if (at::GradMode::is_enabled() && (a.requires_grad() || b.requires_grad())) {
        node = std::shared_ptr<LinearNode>(new LinearNode(), torch::autograd::deleteNode);
        node->lin = &linear_of(name, kind);
        node->kind = kind;
        node->has_order = order.has_value();
        node->a = torch::autograd::SavedVariable(a, false);
        node->b = torch::autograd::SavedVariable(b, false);
        node->offsets = torch::autograd::SavedVariable(offsets, false);
        node->blocks = torch::autograd::SavedVariable(blocks, false);
        if (order) node->order = torch::autograd::SavedVariable(*order, false);
        node->set_next_edges(torch::autograd::collect_next_edges(a, b));
    }
    Tensor out = [&] {
        at::AutoDispatchBelowADInplaceOrView guard;
        return op.call(a, b, order, offsets, blocks, name, kind);
    }();
    if (node) torch::autograd::set_history(out, node);
    return out;
}

thread_local std::string grouped_error;

}  // namespace

TORCH_LIBRARY_FRAGMENT(openequivariance_b200, m) {
    const std::vector<at::Tag> tags{at::Tag::pt2_compliant_tag};
    m.def("row_groups(Tensor index, int groups) -> (Tensor, Tensor, Tensor, Tensor)", tags);
    m.def("row_groups_from_counts(Tensor counts, int rows) -> (Tensor, Tensor, Tensor)", tags);
    m.def("grouped_linear(Tensor a, Tensor b, Tensor? order, Tensor offsets, Tensor blocks, str map, int kind) -> Tensor", tags);
}
TORCH_LIBRARY_IMPL(openequivariance_b200, CUDA, m) {
    m.impl("row_groups", TORCH_FN(row_groups_cuda));
    m.impl("row_groups_from_counts", TORCH_FN(row_groups_from_counts_cuda));
    m.impl("grouped_linear", TORCH_FN(linear_cuda));
}
TORCH_LIBRARY_IMPL(openequivariance_b200, Autograd, m) { m.impl("grouped_linear", TORCH_FN(linear_autograd)); }

extern "C" {

const char* oeq_torch_grouped_error() { return grouped_error.c_str(); }

// Makes a map known to the ops, so that what cannot be made is refused before a call: an OEQ code, or -1 (oeq_torch_grouped_error).
int oeq_torch_grouped_register(const char* name) {
    try {
        const Linear* lin = nullptr;
        return find_linear(name, lin);
    } catch (const std::exception& e) {
        grouped_error = e.what();
        return -1;
    }
}

}  // extern "C"
