// Drafted tokens and log probabilities: DraftBatch, ops.accept_draft, ops.token_log_probs.  They check and unwrap the tensors and
// call the C ABI on torch's current stream.
#include "draft.h"

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>
#include <torch/extension.h>

#include <algorithm>
#include <atomic>
#include <cstring>
#include <stdexcept>

#include "token_lists.h"

namespace py = pybind11;

namespace ca_host {

namespace {
void need(bool ok, const std::string& msg) {
    if (!ok) throw std::runtime_error(msg);
}
void check_rc(int rc, const char* what) {
    if (rc != CA_OK) throw std::runtime_error(std::string(what) + ": " + ca_last_error());
}
}  // namespace

torch::Tensor scratch_on(torch::Device device, c10::ScalarType type, int64_t n) { return at::detail::empty_cuda({n}, type, device, c10::nullopt); }

torch::Tensor part_of(const torch::Tensor& whole, c10::ScalarType type, int64_t at, c10::IntArrayRef sizes) {
    torch::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(whole.storage()), whole.key_set(), c10::scalarTypeToTypeMeta(type));
    t.unsafeGetTensorImpl()->set_storage_offset(at);
    t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
    return t;
}

bool capturing(torch::Device device) {
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    const cudaError_t e = cudaStreamIsCapturing(c10::cuda::getCurrentCUDAStream(device.index()).stream(), &st);
    return e != cudaSuccess || st != cudaStreamCaptureStatusNone;
}

Uploaded::Uploaded(const std::vector<int32_t>& data, torch::Device device, const char* what) {
    // a captured copy would read the pinned buffer again at every replay, when it is gone
    if (device.is_cuda() && capturing(device)) throw std::runtime_error(std::string(what) + ": not while a graph is being captured: run the step once before");
    torch::Tensor host = torch::empty({(int64_t)data.size()}, torch::TensorOptions().dtype(torch::kInt32).pinned_memory(device.is_cuda()));
    std::memcpy(host.data_ptr(), data.data(), data.size() * sizeof(int32_t));
    if (!device.is_cuda()) {
        tensor_ = host;
        return;
    }
    c10::cuda::CUDAGuard guard(device);
    tensor_ = host.to(device, torch::kInt32, /*non_blocking=*/true);
    const auto stream = c10::cuda::getCurrentCUDAStream(device.index());
    stream_ = stream.id();
    ready_ = std::make_shared<at::cuda::CUDAEvent>();
    ready_->record(stream);
}

const int32_t* Uploaded::use() {
    if (ready_) {
        const auto stream = c10::cuda::getCurrentCUDAStream(tensor_.device().index());
        // a stream that is being captured cannot wait for an event of before; capturing begins on an idle device
        if (stream.id() != stream_ && !capturing(tensor_.device())) {
            c10::cuda::CUDAGuard guard(tensor_.device());
            ready_->block(stream);
            c10::cuda::CUDACachingAllocator::recordStream(tensor_.storage().data_ptr(), stream);
        }
    }
    return tensor_.data_ptr<int32_t>();
}

DraftBatch::DraftBatch(const std::vector<std::vector<int>>& trees, torch::Device device) : device_(device) {
    static std::atomic<int64_t> made{0};
    serial_ = ++made;
    if (device_.is_cuda() && !device_.has_index()) device_ = torch::Device(torch::kCUDA, c10::cuda::current_device());
    first_.push_back(0);
    int64_t total = 0;
    size_t most = 0;
    for (const auto& t : trees) {
        need(t.size() <= CA_DRAFT_MAX_NODES, "DraftBatch: a tree has more than " + std::to_string(CA_DRAFT_MAX_NODES) + " nodes");
        int roots = 0;
        for (size_t i = 0; i < t.size(); i++) {
            need(t[i] >= -1 && t[i] < (int)i, "DraftBatch: a node's parent must be a node before it, or -1");
            roots += t[i] < 0;
        }
        rooted_ = rooted_ && roots <= 1;
        total += (int64_t)t.size();
        need(total < (1 << 30), "DraftBatch: too many nodes");
        most = std::max(most, t.size());
        first_.push_back((int32_t)total);
    }
    words_ = std::max<int>(2, (int)(most + 63) / 64 * 2);
    // seen first: it is read 8 bytes at a time
    const int64_t T = total, R = (int64_t)trees.size();
    const int64_t at_row = T * words_ + 2 * T;
    at_parent_ = T * words_;
    at_depth_ = at_parent_ + T;
    at_first_ = at_row + T;
    std::vector<int32_t> data((size_t)std::max<int64_t>(1, at_first_ + R + 1), 0);
    depths_.resize((size_t)T);
    for (int64_t r = 0; r < R; r++) {
        const auto& t = trees[(size_t)r];
        for (size_t i = 0; i < t.size(); i++) {
            const int64_t n = first_[(size_t)r] + (int64_t)i;
            uint32_t* line = reinterpret_cast<uint32_t*>(data.data()) + n * words_;
            if (t[i] >= 0) {
                const int64_t up = first_[(size_t)r] + t[i];
                std::memcpy(line, reinterpret_cast<uint32_t*>(data.data()) + up * words_, (size_t)words_ * 4);
                depths_[(size_t)n] = depths_[(size_t)up] + 1;
            }
            line[i / 32] |= 1u << (i % 32);
            max_depth_ = std::max(max_depth_, (int)depths_[(size_t)n]);
            data[(size_t)(at_parent_ + n)] = t[i];
            data[(size_t)(at_depth_ + n)] = depths_[(size_t)n];
            data[(size_t)(at_row + n)] = (int32_t)r;
        }
    }
    std::copy(first_.begin(), first_.end(), data.begin() + at_first_);
    buffer_ = Uploaded(data, device_, "DraftBatch");
    const torch::Tensor b = buffer_.tensor();
    parents = b.narrow(0, at_parent_, T);
    depths = b.narrow(0, at_depth_, T);
    row_of = b.narrow(0, at_row, T);
}

DraftBatch::View DraftBatch::view(std::vector<torch::Tensor>* keep) {
    const int32_t* p = buffer_.use();
    if (keep && device_.is_cuda() && capturing(device_)) keep->push_back(buffer_.tensor());
    return {p + at_first_, p + at_parent_, p + at_depth_, reinterpret_cast<const uint32_t*>(p)};
}

namespace {

using torch::Tensor;

bool i32_vec(const Tensor& t, torch::Device d, int64_t n) {
    return t.device() == d && t.scalar_type() == torch::kInt32 && t.dim() == 1 && t.is_contiguous() && t.numel() == n;
}
bool f32_vec(const Tensor& t, torch::Device d, int64_t n) {
    return t.device() == d && t.scalar_type() == torch::kFloat32 && t.dim() == 1 && t.is_contiguous() && t.numel() == n;
}

py::tuple accept_draft(DraftBatch& draft, Tensor tokens, Tensor choice, c10::optional<Tensor> log_probs, c10::optional<Tensor> entropy, double epsilon,
                       double delta) {
    const torch::Device dev = draft.device();
    const int64_t n = draft.n_nodes(), rows = draft.n_rows();
    need(dev.is_cuda(), "accept_draft: a draft on a CUDA device is required (there is no CPU path)");
    need(draft.rooted(), "accept_draft: every tree must have one node without a parent");
    need(i32_vec(tokens, dev, n) && i32_vec(choice, dev, n), "accept_draft: tokens and choice must be contiguous int32 [n_nodes] on the draft's device");
    need(log_probs.has_value() == entropy.has_value(), "accept_draft: log_probs and entropy come together");
    if (log_probs.has_value()) {
        need(f32_vec(*log_probs, dev, n) && f32_vec(*entropy, dev, n), "accept_draft: log_probs and entropy must be contiguous fp32 [n_nodes] on the draft's device");
        need(epsilon > 0 && delta > 0, "accept_draft: epsilon and delta must be positive");
    }
    c10::cuda::CUDAGuard guard(dev);
    const int64_t width = draft.max_depth() + 1;
    const Tensor out = scratch_on(dev, torch::kInt32, rows * (width + 2));
    Tensor path = part_of(out, torch::kInt32, 0, {rows, width}), count = part_of(out, torch::kInt32, rows * width, {rows}),
           next = part_of(out, torch::kInt32, rows * (width + 1), {rows});
    const auto view = draft.view();
    ca_accept_args a{};
    a.first = view.first;
    a.parent = view.parent;
    a.depth = view.depth;
    a.seen = view.seen;
    a.words = draft.words();
    a.n_rows = (int32_t)rows;
    a.width = (int32_t)width;
    a.tokens = tokens.data_ptr<int32_t>();
    a.choice = choice.data_ptr<int32_t>();
    a.log_probs = log_probs.has_value() ? log_probs->data_ptr<float>() : nullptr;
    a.entropy = entropy.has_value() ? entropy->data_ptr<float>() : nullptr;
    a.epsilon = epsilon;
    a.delta = delta;
    int32_t* o = out.data_ptr<int32_t>();
    a.path = o;
    a.count = o + rows * width;
    a.next = o + rows * (width + 1);
    check_rc(ca_accept_draft(&a, c10::cuda::getCurrentCUDAStream(dev.index()).stream()), "accept_draft");
    return py::make_tuple(path, count, next);
}

py::tuple token_log_probs(Tensor logits, c10::optional<Tensor> tokens, c10::optional<Tensor> rows, int64_t top) {
    need(logits.is_cuda() && logits.dim() == 2 && logits.size(1) >= 1 && (logits.stride(1) == 1 || logits.size(1) == 1),
         "token_log_probs: logits must be [n_rows, vocab] with contiguous rows on a CUDA device (there is no CPU path)");
    const auto st = logits.scalar_type();
    need(st == torch::kFloat16 || st == torch::kFloat32 || st == torch::kBFloat16, "token_log_probs: fp16, bf16 and fp32 logits only");
    const torch::Device dev = logits.device();
    const int64_t n = logits.size(0), vocab = logits.size(1);
    need(vocab < (int64_t(1) << 31) && n < (int64_t(1) << 31), "token_log_probs: too many rows or tokens");
    need(top >= 0 && top <= CA_MAX_TOP && top <= vocab, "token_log_probs: top must be 0 to " + std::to_string(CA_MAX_TOP) + " and not above the vocabulary");
    need(tokens.has_value() || !rows.has_value(), "token_log_probs: rows name the rows of tokens");
    int64_t asked = 0;
    if (tokens.has_value()) {
        asked = tokens->numel();
        need(i32_vec(*tokens, dev, asked) && asked < (int64_t(1) << 31), "token_log_probs: tokens must be contiguous int32 [n_tokens] on the logits' device");
        if (rows.has_value()) need(i32_vec(*rows, dev, asked), "token_log_probs: rows must be contiguous int32 [n_tokens] on the logits' device");
        else need(asked == n, "token_log_probs: one token per row is required (or rows)");
    }
    c10::cuda::CUDAGuard guard(dev);
    const Tensor out = scratch_on(dev, torch::kFloat32, asked + n + 2 * n * top);
    Tensor log_probs = part_of(out, torch::kFloat32, 0, {asked}), entropy = part_of(out, torch::kFloat32, asked, {n}),
           top_lp = part_of(out, torch::kFloat32, asked + n, {n, top}), top_ids = part_of(out, torch::kInt32, asked + n + n * top, {n, top});
    ca_log_probs_args a{};
    a.dtype = st == torch::kFloat16 ? CA_DTYPE_F16 : (st == torch::kFloat32 ? CA_DTYPE_F32 : CA_DTYPE_BF16);
    const Tensor scratch = scratch_on(dev, torch::kUInt8, std::max<int64_t>(1, ca_log_probs_scratch((int)n, (int)vocab, a.dtype, (int)top)));
    a.logits = logits.data_ptr();
    a.row_stride = n > 1 ? logits.stride(0) : vocab;
    a.n_rows = (int32_t)n;
    a.vocab = (int32_t)vocab;
    a.tokens = tokens.has_value() ? tokens->data_ptr<int32_t>() : nullptr;
    a.rows = rows.has_value() ? rows->data_ptr<int32_t>() : nullptr;
    a.n_tokens = (int32_t)asked;
    a.top = (int32_t)top;
    a.log_probs = log_probs.data_ptr<float>();
    a.entropy = entropy.data_ptr<float>();
    a.top_log_probs = top_lp.data_ptr<float>();
    a.top_ids = top_ids.data_ptr<int32_t>();
    a.scratch = scratch.data_ptr();
    check_rc(ca_token_log_probs(&a, c10::cuda::getCurrentCUDAStream(dev.index()).stream()), "token_log_probs");
    return py::make_tuple(log_probs, entropy, top_lp, top_ids);
}

}  // namespace

void init_draft(py::module& m, py::module& ops) {
    py::class_<DraftBatch, std::shared_ptr<DraftBatch>>(m, "DraftBatch", py::module_local())
      .def(py::init([](const std::vector<std::vector<int>>& parents, py::object device) {
               if (py::isinstance<py::str>(device)) device = py::module_::import("torch").attr("device")(device);
               return std::make_shared<DraftBatch>(parents, torch::python::detail::py_object_to_device(device));
           }),
           py::arg("parents"), py::arg("device"))
      .def_property_readonly("n_rows", &DraftBatch::n_rows)
      .def_property_readonly("n_nodes", &DraftBatch::n_nodes)
      .def_property_readonly("max_depth", &DraftBatch::max_depth)
      .def_property_readonly("first", &DraftBatch::first)
      .def_readonly("depths", &DraftBatch::depths)
      .def_readonly("row_of", &DraftBatch::row_of)
      .def_readonly("parents", &DraftBatch::parents);
    ops.def("accept_draft", &accept_draft, py::arg("draft"), py::arg("tokens"), py::arg("choice"), py::arg("log_probs") = py::none(),
            py::arg("entropy") = py::none(), py::arg("epsilon") = 0.09, py::arg("delta") = 0.3,
            "(path [n_rows, max_depth + 1], count, next): of every tree the deepest node whose line is accepted");
    ops.def("token_log_probs", &token_log_probs, py::arg("logits"), py::arg("tokens") = py::none(), py::arg("rows") = py::none(), py::arg("top") = 0,
            "(log probabilities of tokens, entropy of the rows, log probabilities and ids of the top best tokens)");
}

}  // namespace ca_host
