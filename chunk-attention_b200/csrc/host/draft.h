// DraftBatch — a tree of drafted tokens for every row of a cache, as the kernels read it: one pinned buffer, one upload.
#pragma once
#include <ATen/cuda/CUDAEvent.h>
#include <torch/torch.h>

#include <vector>

#include "../../../include/chunk_attn_b200.h"

namespace ca_host {

// A device buffer made on one stream and read on others
class Uploaded {
  public:
    Uploaded() = default;
    Uploaded(const std::vector<int32_t>& data, torch::Device device, const char* what);
    bool defined() const { return tensor_.defined(); }
    // the buffer for work on the current stream of its device, which waits for the upload and keeps the buffer
    const int32_t* use();
    torch::Tensor tensor() const { return tensor_; }

  private:
    torch::Tensor tensor_;
    std::shared_ptr<at::cuda::CUDAEvent> ready_;
    c10::StreamId stream_ = 0;
};
// Outputs and scratch without the way through torch's dispatcher (accept_draft 8.2 -> 5.1 us a call, token_log_probs 9.0 -> 5.5 us of the host): a
// tensor of n elements, and one over a part of another's memory, from element `at` of its own type on
torch::Tensor scratch_on(torch::Device device, c10::ScalarType type, int64_t n);
torch::Tensor part_of(const torch::Tensor& whole, c10::ScalarType type, int64_t at, c10::IntArrayRef sizes);
bool capturing(torch::Device device);  // whether the current stream is being captured into a graph

class DraftBatch {
  public:
    // parents[r][i]: the node above node i of row r's tree (a lower number), -1: none, its parent is the row's last cached token
    DraftBatch(const std::vector<std::vector<int>>& parents, torch::Device device);

    int n_rows() const { return (int)first_.size() - 1; }
    int n_nodes() const { return first_.back(); }
    int max_depth() const { return max_depth_; }  // -1: no nodes
    bool rooted() const { return rooted_; }       // no tree has two nodes without a parent
    const std::vector<int32_t>& first() const { return first_; }
    const std::vector<int32_t>& host_depths() const { return depths_; }
    int64_t serial() const { return serial_; }
    torch::Device device() const { return device_; }
    int words() const { return words_; }

    // int32 views of the uploaded buffer: position of every node above its row's cached tokens, its row, its parent within the tree
    torch::Tensor depths, row_of, parents;

    // addresses for work on the current stream; `keep` gets the buffer when the stream is being captured
    struct View { const int32_t *first, *parent, *depth; const uint32_t* seen; };
    View view(std::vector<torch::Tensor>* keep = nullptr);

  private:
    std::vector<int32_t> first_, depths_;
    torch::Device device_;
    Uploaded buffer_;
    int64_t serial_;
    int64_t at_first_ = 0, at_parent_ = 0, at_depth_ = 0;
    int words_ = 2, max_depth_ = -1;
    bool rooted_ = true;
};

}  // namespace ca_host
