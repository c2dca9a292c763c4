// Attention of drafted tokens: the work list of a step (host) and the parameters of its kernels.
//
// A row of the cache brings a TREE of drafted tokens ("nodes"): node i sees every cached token of its row, its ancestors in the
// tree and itself.  Drafted keys and values are operands, not part of the pool: a prefix tree only ever holds accepted tokens.
//
// The cached part is walked as decode steps walk it: chunks that the same rows share form a run, which is read once for the nodes of
// all these rows, and the other chunks of a row are its private part, which also takes the row's tree.  A unit (a run, or a private part) times a
// block of its nodes is cut along its tokens into ITEMS.  An item is the same for all heads; the kernels expand it over the
// key/value heads, whose query heads are the columns of a node.  A node that one item serves whole is stored by it; the others' partial
// results (running maximum, sum, un-normalised O) are combined by a second kernel.
#pragma once
#include <stdint.h>

#include <string>
#include <vector>

#if defined(__CUDACC__)
#include <cuda_runtime.h>
#endif

#include "../../include/chunk_attn_b200.h"
#include "ca_layout.h"

namespace ca {

struct DraftItem {
    int32_t node0, n_nodes;  // the block of nodes
    int32_t list, n_tiles;   // its chunks: {pool slot, tokens} pairs from tiles[2 * list] on
    int32_t slot;            // partial results go to slots slot .. slot + n_nodes - 1; -1: finished rows are stored
    int32_t tree, n_drafted; // first node of the row's tree and how many of its nodes the block may see; 0: none
    int32_t tokens;          // of all its tiles
    int32_t head[8];         // its first four {pool slot, tokens} pairs once more: a CTA's first copies need not wait for the list
};
static_assert(sizeof(DraftItem) == 64, "DraftItem is read on the device as four int4");

struct DraftPlan {
    std::vector<DraftItem> items;  // longest first
    std::vector<int32_t> tiles;
    std::vector<int32_t> merge_nodes, merge_off{0}, merge_slots;
    int32_t n_slots = 0;
    int32_t n_nodes = 0, block_nodes = 1;
    // everything of it that kernels read, in one array for one upload (16-byte aligned parts)
    std::vector<int32_t> data;
    int64_t at_tiles = 0, at_nodes = 0, at_off = 0, at_slots = 0;
};

struct DraftPlanShape {
    int chunk_size = 64, tpp_threshold = 1;
    int64_t max_chunks = 0;
    int kv_heads = 1, group = 1;
    int block_rows = 128;  // query rows of an item at most (at least one node's)
    int ctas = 296;        // CTAs that run at a time
};
// first[0 .. n_rows]: first node of every row's tree.  An empty string, or why the input was rejected.
std::string build_draft_plan(DraftPlan& plan, const ca_chunk_info* infos, int n_infos, const int32_t* first, int n_rows, const DraftPlanShape& shape);

#if defined(__CUDACC__)
struct DraftParams {
    const void* pool;
    Geometry geo;              // n_heads: key/value heads
    int group;                 // query heads per key/value head
    int d_key, d_value;        // of q, k, v and out; the pool's may be padded
    const void *q, *k, *v;     // [n_nodes, heads, .]: element strides below, the last 1
    int64_t q_node, q_head, k_node, k_head, v_node, v_head;
    bool whole_granules;       // addresses, strides and head sizes of k and v are whole 16-byte units
    void* out;                 // [n_nodes, heads, d_value]
    float scale_log2;          // scale * log2(e)
    int sink;
    const uint32_t* seen;      // [n_nodes][words]: bit j: node j of the tree is the node itself or above it
    int words;
    const DraftItem* items;
    int n_items, n_nodes;
    const int32_t* tiles;
    float* part_o;             // [n_slots][heads][part_width]
    float2* part_ml;           // [n_slots][heads]: running maximum (log2 units), sum
    int part_width;
    const int32_t *merge_nodes, *merge_off, *merge_slots;
    int n_merge, n_merge_slots;
    int n_list, n_slots;       // entries of tiles, partial slots
    int max_chunks;
    int* status;
    long long wait_limit;
    int dependent;             // CA_OPT_DEPENDENT_LAUNCH
    bool settled;              // the work list and seen may be read while the kernel before runs
};
// First of all in every kernel: unless nothing that still runs writes the work list and seen, wait for the kernels before
__device__ __forceinline__ void draft_lists_wait(const DraftParams& p) {
    if (!p.settled) asm volatile("griddepcontrol.wait;" ::: "memory");
}
// What the lists hold may have been written after the kernel began, before its wait: plain loads, which stay behind it
template <typename T> __device__ __forceinline__ T list_load(const T* p) { return *p; }
// nothing in a work list is trusted
__device__ __forceinline__ bool draft_item_ok(const DraftParams& p, int4 a, int4 b, int block_rows) {
    return a.x >= 0 && a.y > 0 && a.x + a.y <= p.n_nodes && a.y * p.group <= block_rows && a.z >= 0 && a.w >= 0 && a.z + a.w <= p.n_list &&
           b.x + a.y <= p.n_slots + (b.x < 0 ? a.y : 0) && b.y >= 0 && b.z >= 0 && b.y + b.z <= p.n_nodes && b.z <= 32 * p.words && a.w + b.z > 0;
}
#endif
// query rows of an item that the any-geometry kernel takes, for units of so many
inline int draft_generic_rows(int unit_rows) { return unit_rows <= 4 ? 4 : (unit_rows <= 16 ? (unit_rows + 3) / 4 * 4 : (unit_rows <= 32 ? 32 : 64)); }

#if defined(__CUDACC__)
int draft_generic_ctas(int block_rows, int dk, int dv, int esize);  // that run at a time
cudaError_t launch_draft_generic(const DraftParams& p, int block_rows, int dtype, cudaStream_t stream);
bool draft_tc_serves(const Geometry& g, int d_key, int d_value, int group, float scale);
cudaError_t launch_draft_tc(const DraftParams& p, int dtype, cudaStream_t stream);
constexpr int DRAFT_TC_ROWS = 128;  // query rows of an item
cudaError_t launch_draft_merge(const DraftParams& p, int dtype, cudaStream_t stream);

struct AcceptParams {
    const int32_t* first;      // [n_rows + 1]
    const int32_t* parent;     // [n_nodes], within the tree, -1: none
    const int32_t* depth;      // [n_nodes]
    const uint32_t* seen;      // [n_nodes][words]
    int words, n_rows, width;  // width: entries of a path
    const int32_t *tokens, *choice;
    const float *log_probs, *entropy;  // null: greedy
    float log_epsilon, log_delta;
    int32_t *path, *count, *next;
};
cudaError_t launch_accept_draft(const AcceptParams& p, cudaStream_t stream);
#endif

}  // namespace ca
