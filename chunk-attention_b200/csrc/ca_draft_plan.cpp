// Host-side work list of attention over drafted trees; see ca_draft.h.
#include "ca_draft.h"

#include <algorithm>

namespace ca {
namespace {

// What an item costs beside its tokens, in tokens of its tiles, and what it costs more when its rows have to be combined with other
// items': set-up, queries and epilogue of a CTA, then partial rows out and in and the second kernel.
constexpr int ITEM_TOKENS = 96, PARTIAL_TOKENS = 96;

struct Unit {
    std::vector<int32_t> tiles;  // {chunk, tokens}
    int32_t tokens = 0;
    int32_t node0 = 0, n_nodes = 0;
    int32_t tree = 0, n_tree = 0;  // of a private part
    int32_t blocks(int per_block) const { return (n_nodes + per_block - 1) / per_block; }
};

}  // namespace

std::string build_draft_plan(DraftPlan& plan, const ca_chunk_info* infos, int n_infos, const int32_t* first, int n_rows, const DraftPlanShape& s) {
    plan = DraftPlan();
    if (n_rows < 0 || n_infos < 0 || !first || (n_infos > 0 && !infos)) return "draft plan: null or negative input";
    if (s.chunk_size <= 0 || s.kv_heads <= 0 || s.group <= 0 || s.block_rows <= 0 || s.ctas <= 0) return "draft plan: bad sizes";
    for (int r = 0; r < n_rows; r++)
        if (first[r + 1] < first[r] || first[0] != 0) return "draft plan: the first nodes of the rows' trees must not fall";
    plan.n_nodes = n_rows > 0 ? first[n_rows] : 0;
    plan.block_nodes = std::max(1, s.block_rows / s.group);
    if (plan.n_nodes == 0) return "";

    // ---- units: runs of shared chunks, then every row's private part
    std::vector<Unit> units;
    std::vector<Unit> own((size_t)n_rows);
    int run_b = -1, run_e = -1;
    for (int i = 0; i < n_infos; i++) {
        const ca_chunk_info& ci = infos[i];
        if (ci.chunk_id < 0 || ci.chunk_id >= s.max_chunks) return "draft plan: chunk id outside the pool";
        if (ci.n_tokens < 0 || ci.n_tokens > s.chunk_size) return "draft plan: token count outside the chunk";
        if (ci.seq_begin < 0 || ci.seq_end > n_rows || ci.seq_begin >= ci.seq_end) return "draft plan: row range outside the batch";
        const int n_nodes = first[ci.seq_end] - first[ci.seq_begin];
        if (ci.n_tokens == 0 || n_nodes == 0) continue;
        if (ci.seq_end - ci.seq_begin > std::max(1, s.tpp_threshold)) {
            // depth-first order: a chain of chunks with the same rows follows one another
            if (units.empty() || run_b != ci.seq_begin || run_e != ci.seq_end) {
                units.emplace_back();
                units.back().node0 = first[ci.seq_begin];
                units.back().n_nodes = n_nodes;
                run_b = ci.seq_begin;
                run_e = ci.seq_end;
            }
            units.back().tiles.insert(units.back().tiles.end(), {ci.chunk_id, ci.n_tokens});
            units.back().tokens += ci.n_tokens;
        } else {
            for (int r = ci.seq_begin; r < ci.seq_end; r++) {
                own[r].tiles.insert(own[r].tiles.end(), {ci.chunk_id, ci.n_tokens});
                own[r].tokens += ci.n_tokens;
            }
        }
    }
    const size_t n_runs = units.size();
    for (int r = 0; r < n_rows; r++) {
        Unit& u = own[r];
        u.node0 = u.tree = first[r];
        u.n_nodes = u.n_tree = first[r + 1] - first[r];
        if (u.n_nodes > 0) units.push_back(std::move(u));
    }
    // how many units serve a node
    std::vector<int32_t> served((size_t)plan.n_nodes, 0);
    for (const Unit& u : units)
        for (int n = 0; n < u.n_nodes; n++) served[u.node0 + n]++;

    // ---- the length of a piece: the one whose items, as many at a time as CTAs fit, are done soonest
    int longest = 1;
    for (const Unit& u : units) longest = std::max(longest, u.tokens + u.n_tree);
    auto pieces_of = [&](const Unit& u, int len) {
        const int chunks = (int)u.tiles.size() / 2;
        return std::max(1, std::min((u.tokens + u.n_tree + len - 1) / len, chunks));
    };
    int best_len = longest;
    double best_cost = 0;
    for (int p = 1; p <= 64; p++) {
        const int len = std::max(s.chunk_size, (longest + p - 1) / p);
        double sum = 0, most = 0, n_items = 0;
        for (const Unit& u : units) {
            const int pieces = pieces_of(u, len);
            const bool partial = pieces > 1 || served[u.node0] > 1;
            const double each = (double)(u.tokens + u.n_tree) / pieces + ITEM_TOKENS + (partial ? PARTIAL_TOKENS : 0);
            const double n = (double)pieces * u.blocks(plan.block_nodes) * s.kv_heads;
            sum += n * each;
            n_items += n;
            most = std::max(most, each);
        }
        const double cost = n_items <= s.ctas ? most : std::max(most, sum / s.ctas + 0.5 * most);
        if (p == 1 || cost < 0.97 * best_cost) {
            best_len = len;
            best_cost = cost;
        }
        if (len == s.chunk_size) break;
    }

    // ---- items
    std::vector<std::vector<int32_t>> slots_of((size_t)plan.n_nodes);
    for (size_t ui = 0; ui < units.size(); ui++) {
        const Unit& u = units[ui];
        const int chunks = (int)u.tiles.size() / 2, pieces = pieces_of(u, best_len), blocks = u.blocks(plan.block_nodes);
        const int list = (int)plan.tiles.size() / 2;
        plan.tiles.insert(plan.tiles.end(), u.tiles.begin(), u.tiles.end());
        for (int pc = 0; pc < pieces; pc++) {
            // equal shares of the chunks; the tree goes with the last one
            const int c0 = (int)((int64_t)chunks * pc / pieces), c1 = (int)((int64_t)chunks * (pc + 1) / pieces);
            for (int b = 0; b < blocks; b++) {
                DraftItem it{};
                it.node0 = u.node0 + (int)((int64_t)u.n_nodes * b / blocks);
                it.n_nodes = u.node0 + (int)((int64_t)u.n_nodes * (b + 1) / blocks) - it.node0;
                it.list = list + c0;
                it.n_tiles = c1 - c0;
                it.tree = u.tree;
                it.n_drafted = ui >= n_runs && pc == pieces - 1 ? it.node0 + it.n_nodes - u.tree : 0;
                for (int c = c0; c < c1; c++) it.tokens += u.tiles[2 * c + 1];
                for (int c = c0; c < std::min(c1, c0 + 4); c++) {
                    it.head[2 * (c - c0)] = u.tiles[2 * c];
                    it.head[2 * (c - c0) + 1] = u.tiles[2 * c + 1];
                }
                it.slot = -1;
                if (pieces > 1 || served[u.node0] > 1) {
                    it.slot = plan.n_slots;
                    plan.n_slots += it.n_nodes;
                    for (int n = 0; n < it.n_nodes; n++) slots_of[it.node0 + n].push_back(it.slot + n);
                }
                plan.items.push_back(it);
            }
        }
    }
    // Longest first, so that the last wave is short; of equal ones the blocks of a piece stay together and find its chunks in L2
    std::stable_sort(plan.items.begin(), plan.items.end(), [](const DraftItem& a, const DraftItem& b) { return a.tokens + a.n_drafted > b.tokens + b.n_drafted; });
    for (int n = 0; n < plan.n_nodes; n++) {
        if (slots_of[n].empty()) continue;
        plan.merge_nodes.push_back(n);
        plan.merge_slots.insert(plan.merge_slots.end(), slots_of[n].begin(), slots_of[n].end());
        plan.merge_off.push_back((int32_t)plan.merge_slots.size());
    }

    auto part = [&](const int32_t* p, size_t n) {
        while (plan.data.size() % 4) plan.data.push_back(0);
        const int64_t at = (int64_t)plan.data.size();
        plan.data.insert(plan.data.end(), p, p + n);
        return at;
    };
    part(reinterpret_cast<const int32_t*>(plan.items.data()), plan.items.size() * (sizeof(DraftItem) / 4));
    plan.at_tiles = part(plan.tiles.data(), plan.tiles.size());
    plan.at_nodes = part(plan.merge_nodes.data(), plan.merge_nodes.size());
    plan.at_off = part(plan.merge_off.data(), plan.merge_off.size());
    plan.at_slots = part(plan.merge_slots.data(), plan.merge_slots.size());
    return "";
}

}  // namespace ca
