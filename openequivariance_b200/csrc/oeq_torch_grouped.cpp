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

#include <deque>
#include <mutex>
#include <optional>
#include <tuple>

#include "oeq_torch_common.h"

namespace {

using at::Tensor;
using oeq_torch::check;
using oeq_torch::direct;
using oeq_torch::index_ptr;

enum Kind { PRODUCT = 0, INPUT = 1, WEIGHTS = 2 };      // F(x, w), T(dz, w), G(x, dz)

// Maps live as long as the process: an autograd graph may hold one after its front end has gone.
struct Linear {
    oeq_grouped* handle;
    int64_t in, out, numel;
    int64_t width(int64_t kind) const { return kind == PRODUCT ? out : (kind == INPUT ? in : numel); }     // of a result
    int64_t width_a(int64_t kind) const { return kind == INPUT ? out : in; }
    int64_t width_b(int64_t kind) const { return kind == WEIGHTS ? out : numel; }
};
std::mutex linear_mutex;
std::deque<Linear>& linears() {
    static auto* d = new std::deque<Linear>();
    return *d;
}
const Linear& linear_of(int64_t id, int64_t kind) {
    std::lock_guard<std::mutex> lock(linear_mutex);
    TORCH_CHECK_VALUE(id >= 0 && id < (int64_t)linears().size() && kind >= PRODUCT && kind <= WEIGHTS, "no such linear map");
    return linears()[id];       // (a deque's elements stay where they are)
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
Tensor linear_cuda(const Tensor& a_in, const Tensor& b_in, const std::optional<Tensor>& order_in, const Tensor& offsets_in, const Tensor& blocks_in,
                   int64_t id, int64_t kind) {
    const Linear& lin = linear_of(id, kind);
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

using Signature = Tensor(const Tensor&, const Tensor&, const std::optional<Tensor>&, const Tensor&, const Tensor&, int64_t, int64_t);

Tensor call_linear(const Tensor& a, const Tensor& b, const std::optional<Tensor>& order, const Tensor& offsets, const Tensor& blocks, int64_t id,
                   int64_t kind) {
    if (direct({a, b, offsets, blocks})) return linear_cuda(a, b, order, offsets, blocks, id, kind);
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("openequivariance_b200::grouped_linear", "").typed<Signature>();
    return op.call(a, b, order, offsets, blocks, id, kind);
}

struct LinearNode final : torch::autograd::Node {
    int64_t id, kind;
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
        auto call = [&](int64_t k, const Tensor& p, const Tensor& q) { return call_linear(p, q, ord, off, blk, id, k); };
        Tensor ga, gb;
        if (task_should_compute_output(0)) ga = kind == PRODUCT ? call(INPUT, e, y) : (kind == INPUT ? call(PRODUCT, e, y) : call(INPUT, y, e));
        if (task_should_compute_output(1)) gb = kind == PRODUCT ? call(WEIGHTS, x, e) : (kind == INPUT ? call(WEIGHTS, e, x) : call(PRODUCT, x, e));
        return {ga, gb};
    }
};

Tensor linear_autograd(const Tensor& a, const Tensor& b, const std::optional<Tensor>& order, const Tensor& offsets, const Tensor& blocks, int64_t id,
                       int64_t kind) {
    TORCH_CHECK_NOT_IMPLEMENTED(!torch::autograd::isFwGradDefined(a) && !torch::autograd::isFwGradDefined(b),
                                "openequivariance_b200: the operators have no forward-mode derivative");
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("openequivariance_b200::grouped_linear", "").typed<Signature>();
    std::shared_ptr<LinearNode> node;
    if (at::GradMode::is_enabled() && (a.requires_grad() || b.requires_grad())) {
        node = std::shared_ptr<LinearNode>(new LinearNode(), torch::autograd::deleteNode);
        node->id = id;
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
        return op.call(a, b, order, offsets, blocks, id, kind);
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
    m.def("grouped_linear(Tensor a, Tensor b, Tensor? order, Tensor offsets, Tensor blocks, int linear, int kind) -> Tensor", tags);
}
TORCH_LIBRARY_IMPL(openequivariance_b200, CUDA, m) {
    m.impl("row_groups", TORCH_FN(row_groups_cuda));
    m.impl("row_groups_from_counts", TORCH_FN(row_groups_from_counts_cuda));
    m.impl("grouped_linear", TORCH_FN(linear_cuda));
}
TORCH_LIBRARY_IMPL(openequivariance_b200, Autograd, m) { m.impl("grouped_linear", TORCH_FN(linear_autograd)); }

extern "C" {

const char* oeq_torch_grouped_error() { return grouped_error.c_str(); }

// Makes a map known to the ops: its number, or -1.
int64_t oeq_torch_grouped_register(oeq_grouped* handle, int64_t in, int64_t out) {
    try {
        std::lock_guard<std::mutex> lock(linear_mutex);
        linears().push_back({handle, in, out, oeq_grouped_weight_numel(handle)});
        return (int64_t)linears().size() - 1;
    } catch (const std::exception& e) {
        grouped_error = e.what();
        return -1;
    }
}

}  // extern "C"
