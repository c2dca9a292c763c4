// Attention of drafted trees in any geometry and type (fp32 arithmetic on CUDA cores), the combination of partial results, and the
// walk that accepts drafted tokens.
//
// For node i of row r with query q, over the cached tokens C(r) of its row and its line A(i) (its ancestors and itself):
//   s_j = scale q . k_j,  m = max s_j,  l = sum e^(s_j - m),  out = sum e^(s_j - m) v_j / l,   j in C(r) u A(i)
// (sink: one more score of 0 without a value).  A piece of the keys yields (m, l, un-normalised out); pieces combine by
// out = sum 2^(m_p - M) O_p / sum 2^(m_p - M) l_p, with maxima in log2 units.
#include <algorithm>

#include "ca_draft.h"
#include "ca_draft_row.cuh"
#include "ca_kernels.h"
#include "ca_launch.cuh"
#include "ca_ptx.cuh"
#include "ca_types.cuh"

namespace ca {
namespace {

constexpr int G_THREADS = 256, G_WARPS = 8, G_TOK = 32, G_STAGES = 2;
constexpr float G_NEG_BIG = -1.0e30f;

__host__ __device__ constexpr int whole(int x, int unit) { return (x + unit - 1) / unit * unit; }
struct GenericSizes {
    int k_bytes, v_bytes, q_floats;  // of a key and a value as staged, of a query row
    __host__ __device__ int stage() const { return G_TOK * (k_bytes + v_bytes); }
};
__host__ __device__ inline GenericSizes generic_sizes(int dk, int dv, int esize) { return {whole(dk * esize, 16), whole(dv * esize, 16), whole(dk, 16 / esize)}; }
// Byte of granule g of token t of a staged tile: as the pool has it, 128-byte panels of which the granules of a line are XORed with the token (so
// neither eight tokens' like granules nor a token's granules meet a bank twice), or rows
__device__ __forceinline__ int staged(int t, int g, int row_bytes, int swz) { return swz ? ((g >> 3) * G_TOK + t) * 128 + (((g & 7) ^ (t & 7)) << 4) : t * row_bytes + g * 16; }

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// The tiles of an item: parts of chunks of up to 32 tokens, then of the row's tree
struct Tile { int chunk, first, n; };  // chunk < 0: drafted; n = 0: there is none
template <typename T> struct Walk {
    static constexpr int E = 16 / sizeof(T);
    const DraftParams& p;
    const GenericSizes& z;
    const DraftItem& it;
    const int kvh;
    uint8_t* const stages;
    int j = 0, t0 = 0, d0 = 0, chunk = -1, in_chunk = 0;
    int2 next;  // chunk j's pair, asked for a chunk ahead
    __device__ __forceinline__ int2 entry(int i) const { return i < it.n_tiles ? list_load(reinterpret_cast<const int2*>(p.tiles) + it.list + i) : make_int2(-1, 0); }
    __device__ __forceinline__ Walk(const DraftParams& p, const GenericSizes& z, const DraftItem& it, int kvh, uint8_t* stages, int2 first) : p(p), z(z), it(it), kvh(kvh), stages(stages), next(first) {}
    __device__ __forceinline__ Tile take() {
        while (j < it.n_tiles) {
            if (t0 == 0) {
                chunk = next.x;
                in_chunk = next.y;
                next = entry(j + 1);
                if (chunk < 0 || chunk >= p.max_chunks || in_chunk > p.geo.chunk_size) {
                    if (threadIdx.x == 0) atomicCAS(p.status, STATUS_OK, STATUS_BAD_WORK_LIST);
                    in_chunk = 0;
                }
            }
            if (t0 >= in_chunk) {
                j++;
                t0 = 0;
                continue;
            }
            const Tile t = {chunk, t0, min(G_TOK, in_chunk - t0)};
            t0 += G_TOK;
            return t;
        }
        const Tile t = {-1, d0, max(0, min(G_TOK, it.n_drafted - d0))};
        d0 += G_TOK;
        return t;
    }
    // By a whole block.  Parts of chunks whose rows are whole granules by bulk copies of warp 0, which complete on the stage's barrier (true);
    // drafted rows of whole granules by asynchronous copies, others by plain ones.  Lines behind the tile's tokens hold anything.
    __device__ __forceinline__ bool fetch(const Tile& t, int stage, uint32_t bar) const {
        uint8_t* const sk = stages + stage * z.stage();
        uint8_t* const sv = sk + G_TOK * z.k_bytes;
        const uint32_t to_k = (uint32_t)__cvta_generic_to_shared(sk), to_v = (uint32_t)__cvta_generic_to_shared(sv);
        if (t.chunk >= 0 && p.geo.epg == E) {
            if (threadIdx.x < 32) {  // a panel or a side to a lane
                const int lane = threadIdx.x, k_parts = p.geo.swz ? z.k_bytes / 128 : 1, v_parts = p.geo.v_swz ? z.v_bytes / 128 : 1;
                if (lane == 0) ptx::mbar_arrive_expect_tx(bar, t.n * (z.k_bytes + z.v_bytes));
                __syncwarp();
                if (lane < k_parts + v_parts) {
                    const bool is_v = lane >= k_parts;
                    const int part = is_v ? lane - k_parts : lane, swz = is_v ? p.geo.v_swz : p.geo.swz, line = swz ? 128 : (is_v ? z.v_bytes : z.k_bytes);
                    const uint8_t* from = static_cast<const uint8_t*>(p.pool) + (tile_base_elems(p.geo, t.chunk, kvh, 0) + (is_v ? p.geo.tile_elems : 0)) * (int)sizeof(T);
                    ptx::bulk_copy_g2s((is_v ? to_v : to_k) + part * (G_TOK * 128), from + ((int64_t)part * p.geo.chunk_size + t.first) * line, t.n * line, bar);
                }
            }
            return true;
        }
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        if (t.chunk < 0 && p.whole_granules) {
            auto side = [&](uint32_t to, const void* base, int64_t node, int64_t head, int row_bytes, int swz) {
                const T* from = static_cast<const T*>(base) + (int64_t)(it.tree + t.first + warp) * node + (int64_t)kvh * head;
                for (int g = lane; g < row_bytes / 16; g += 32)
#pragma unroll
                    for (int i = 0; i < G_TOK / G_WARPS; i++)
                        if (warp + G_WARPS * i < t.n) cp_async16(to + staged(warp + G_WARPS * i, g, row_bytes, swz), from + i * G_WARPS * node + g * E);
            };
            side(to_k, p.k, p.k_node, p.k_head, z.k_bytes, p.geo.swz);
            side(to_v, p.v, p.v_node, p.v_head, z.v_bytes, p.geo.v_swz);
        } else {
            auto side = [&](uint8_t* to, const T* from, int d, int row_bytes, int swz, const Geometry& g, int64_t node) {
                for (int x = warp; x < t.n; x += G_WARPS)
#pragma unroll 4
                    for (int e = lane; e < row_bytes / (int)sizeof(T); e += 32) {
                        const T v = e < d ? (t.chunk >= 0 ? from[tile_elem_offset(g, t.first + x, e)] : from[x * node + e]) : from_f32<T>(0.f);
                        reinterpret_cast<T*>(to + staged(x, e / E, row_bytes, swz))[e % E] = v;
                    }
            };
            const T *kt, *vt;
            if (t.chunk >= 0) {
                kt = static_cast<const T*>(p.pool) + tile_base_elems(p.geo, t.chunk, kvh, 0);
                vt = kt + p.geo.tile_elems;
            } else {
                kt = static_cast<const T*>(p.k) + (int64_t)(it.tree + t.first) * p.k_node + (int64_t)kvh * p.k_head;
                vt = static_cast<const T*>(p.v) + (int64_t)(it.tree + t.first) * p.v_node + (int64_t)kvh * p.v_head;
            }
            side(sk, kt, p.d_key, z.k_bytes, p.geo.swz, tile_side(p.geo, 0), p.k_node);
            side(sv, vt, p.d_value, z.v_bytes, p.geo.v_swz, tile_side(p.geo, 1), p.v_node);
        }
        return false;
    }
};

// What both kernels do around a tile: the stages' barriers, the wait for one
struct Stages {
    uint32_t bars, used = 0, phases = 0;  // bits: the stage's tile comes by bulk copies, the phase its barrier is in
    long long limit;
    int* status;
    template <typename T> __device__ __forceinline__ void fetch(const Walk<T>& walk, const Tile& t, int stage) {
        const bool bulk = walk.fetch(t, stage, bars + 8 * stage);
        used = (used & ~(1u << stage)) | (bulk ? 1u << stage : 0u);
    }
    // The tiles of the stage and of n - 1 behind it are there, for the whole block.  False: a copy did not come in time; status is recorded
    template <int N = 1> __device__ __forceinline__ bool wait(int stage) {
        const uint32_t mine = ((1u << N) - 1) << stage, bulk = used & mine;
        bool ok = true;
        if (bulk != mine) asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
        for (int i = 0; i < N; i++)
            if ((bulk >> (stage + i)) & 1) ok = ok && ptx::mbar_wait_bounded(bars + 8 * (stage + i), (phases >> (stage + i)) & 1, limit);
        phases ^= bulk;
        if (__syncthreads_and(ok)) return true;
        if (threadIdx.x == 0) {
            atomicCAS(status, STATUS_OK, STATUS_FULL_WAIT_TIMEOUT);
            for (int i = 0; i < N; i++)
                if ((bulk >> (stage + i)) & 1 && !ptx::mbar_wait_bounded(bars + 8 * (stage + i), ((phases >> (stage + i)) & 1) ^ 1, limit)) atomicCAS(status, STATUS_OK, STATUS_DRAIN_TIMEOUT);
        }
        return false;
    }
};
__device__ __forceinline__ Stages make_stages(const DraftParams& p, uint64_t* bars, int n = G_STAGES) {
    Stages s;
    s.bars = (uint32_t)__cvta_generic_to_shared(bars);
    s.limit = p.wait_limit;
    s.status = p.status;
    if (threadIdx.x == 0) {
        for (int i = 0; i < n; i++) ptx::mbar_init(s.bars + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    return s;
}
// Query rows row, row + step, ... of an item to shared memory as fp32, their loads side by side
template <typename T, int ROWS> __device__ __forceinline__ void stage_queries(const DraftParams& p, const DraftItem& it, int kvh, float* sq, int q_floats, int n_rows, int rows, int row, int step) {
    const int lane = threadIdx.x & 31;
    const T* from[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        const int r = min(row + step * i, n_rows - 1), at = r / p.group;
        from[i] = static_cast<const T*>(p.q) + (int64_t)(it.node0 + at) * p.q_node + (int64_t)(kvh * p.group + r - at * p.group) * p.q_head;
    }
    for (int e0 = lane; e0 < q_floats; e0 += 128) {
        float x[4][ROWS];
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int i = 0; i < ROWS; i++) x[k][i] = e0 + 32 * k < p.d_key ? to_f32(from[i][e0 + 32 * k]) : 0.f;
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int i = 0; i < ROWS; i++)
                if (e0 + 32 * k < q_floats && row + step * i < rows) sq[(row + step * i) * q_floats + e0 + 32 * k] = x[k][i];
    }
}

// An item for one key/value head.  Eight warps with RW query rows each (row r: query head r % group of node r / group); the keys go by in tiles of
// 32 tokens, staged as they are, the next one on its way.  Scores: a lane has a token, and multiplies its key with the warp's rows (read by all
// lanes at once).  Softmax: over the lanes, the rows' steps side by side.  Output: a lane has the columns 4 lane .. 4 lane + 3 of each 128,
// weights come from shared memory.  For 17 rows and more; bound by fp32 products and the reads that feed them (8 rows of 1000 tokens with 120 query rows
// to each of 8 heads of 80 in bf16: 206 us).
template <typename T, int RW, int COLS>  // COLS: groups of 128 value columns
__global__ void __launch_bounds__(G_THREADS, 2) draft_generic_kernel(const DraftParams p, const GenericSizes z) {
    extern __shared__ __align__(128) uint8_t raw[];
    __shared__ uint64_t bars[G_STAGES];
    constexpr int E = 16 / sizeof(T);
    float* const sq = reinterpret_cast<float*>(raw);     // [8 RW][q_floats]
    float* const sp = sq + G_WARPS * RW * z.q_floats;    // [8 RW][32] weights
    uint8_t* const stages = raw + whole((int)sizeof(float) * G_WARPS * RW * (z.q_floats + G_TOK), 128);
    const int dk = p.d_key, dv = p.d_value, stage_bytes = z.stage();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = p.geo.n_heads, group = p.group, H = G * group;
    const int kvh = blockIdx.x % G;
    draft_lists_wait(p);
    const int4 ia = list_load(reinterpret_cast<const int4*>(p.items + blockIdx.x / G)), ib = list_load(reinterpret_cast<const int4*>(p.items + blockIdx.x / G) + 1),
               ic = list_load(reinterpret_cast<const int4*>(p.items + blockIdx.x / G) + 2);
    const DraftItem it = {ia.x, ia.y, ia.z, ia.w, ib.x, ib.y, ib.z, ib.w, {}};
    if (!draft_item_ok(p, ia, ib, G_WARPS * RW)) {
        if (tid == 0) atomicCAS(p.status, STATUS_OK, STATUS_BAD_WORK_LIST);
        return;
    }
    const int n_rows = it.n_nodes * group, row0 = warp * RW;
    const bool busy = row0 < n_rows;
    const int k_gran = whole(dk, E) / E, v_gran = whole(dv, E) / E;  // of a staged row
    Walk<T> tiles(p, z, it, kvh, stages, make_int2(ic.x, ic.y));
    float m[RW], l[RW], o[RW][COLS * 4];
#pragma unroll
    for (int r = 0; r < RW; r++) {
        m[r] = G_NEG_BIG;
        l[r] = 0.f;
#pragma unroll
        for (int c = 0; c < COLS * 4; c++) o[r][c] = 0.f;
    }
    Stages in = make_stages(p, bars);
    // what the work list names is the kernels' before
    Tile now = tiles.take();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (now.n > 0) in.fetch(tiles, now, 0);
#pragma unroll
    for (int half = 0; half < RW; half += 4) stage_queries<T, 4>(p, it, kvh, sq, z.q_floats, n_rows, G_WARPS * RW, row0 + half, 1);
    for (int stage = 0; now.n > 0; stage ^= 1) {
        if (!in.wait(stage)) return;  // nobody reads the tile before this one any more
        const Tile after = tiles.take();
        if (after.n > 0) in.fetch(tiles, after, stage ^ 1);
        if (busy) {
            const uint8_t* const sk = stages + stage * stage_bytes;
            const uint8_t* const sv = sk + G_TOK * z.k_bytes;
            const bool drafted = now.chunk < 0;
            float s[RW];
#pragma unroll
            for (int r = 0; r < RW; r++) s[r] = 0.f;
#pragma unroll 2
            for (int g = 0; g < k_gran; g++) {
                float k[E];
                Granule<T>::load(reinterpret_cast<const T*>(sk + staged(lane, g, z.k_bytes, p.geo.swz)), k);
#pragma unroll
                for (int r = 0; r < RW; r++)
#pragma unroll
                    for (int e = 0; e < E; e += 4) {
                        const float4 q = *reinterpret_cast<const float4*>(sq + (row0 + r) * z.q_floats + g * E + e);
                        s[r] = fmaf(q.x, k[e], s[r]);
                        s[r] = fmaf(q.y, k[e + 1], s[r]);
                        s[r] = fmaf(q.z, k[e + 2], s[r]);
                        s[r] = fmaf(q.w, k[e + 3], s[r]);
                    }
            }
            uint32_t line[RW];  // tokens of the tile that a row sees
            float high[RW];
#pragma unroll
            for (int r = 0; r < RW; r++) {
                line[r] = now.n == 32 ? 0xffffffffu : (1u << now.n) - 1;
                if (drafted) line[r] &= list_load(p.seen + (int64_t)(it.node0 + min(row0 + r, n_rows - 1) / group) * p.words + now.first / 32);
                s[r] = (line[r] >> lane) & 1 ? s[r] * p.scale_log2 : -INFINITY;
                high[r] = s[r];
            }
#pragma unroll
            for (int off = 16; off >= 1; off >>= 1)
#pragma unroll
                for (int r = 0; r < RW; r++) high[r] = fmaxf(high[r], __shfl_xor_sync(0xffffffffu, high[r], off));
#pragma unroll
            for (int r = 0; r < RW; r++) {
                const float mn = fmaxf(m[r], high[r]), alpha = exp2_approx(m[r] - mn), w = (line[r] >> lane) & 1 ? exp2_approx(s[r] - mn) : 0.f;
                m[r] = mn;
                l[r] = l[r] * alpha + w;  // this lane's tokens only: summed over the lanes at the end
                sp[(row0 + r) * G_TOK + lane] = w;
                if (alpha != 1.f) {
#pragma unroll
                    for (int c = 0; c < COLS * 4; c++) o[r][c] *= alpha;
                }
            }
            __syncwarp();
            auto value = [&](int t, int c, float (&v)[4]) {  // columns 128 c + 4 lane ...
                if (128 * c + 4 * lane < v_gran * E) {
                    const int e = 128 * c + 4 * lane;
                    const Pack<T, 4> x = *reinterpret_cast<const Pack<T, 4>*>(sv + staged(t, e / E, z.v_bytes, p.geo.v_swz) + e % E * (int)sizeof(T));
#pragma unroll
                    for (int i = 0; i < 4; i++) v[i] = to_f32(x.v[i]);
                } else {
                    v[0] = v[1] = v[2] = v[3] = 0.f;
                }
            };
            if (!drafted && now.n == G_TOK) {
#pragma unroll 1
                for (int t = 0; t < G_TOK; t += 4) {
                    float v[4][COLS][4];
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int c = 0; c < COLS; c++) value(t + i, c, v[i][c]);
#pragma unroll
                    for (int r = 0; r < RW; r++) {
                        const float4 w4 = *reinterpret_cast<const float4*>(sp + (row0 + r) * G_TOK + t);
                        const float w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                        for (int i = 0; i < 4; i++)
#pragma unroll
                            for (int c = 0; c < COLS; c++)
#pragma unroll
                                for (int e = 0; e < 4; e++) o[r][4 * c + e] = fmaf(w[i], v[i][c][e], o[r][4 * c + e]);
                    }
                }
            } else {
                // values that a row does not see may be infinite: they are left out, not multiplied by zero
#pragma unroll 1
                for (int t = 0; t < now.n; t++) {
                    float v[COLS][4];
#pragma unroll
                    for (int c = 0; c < COLS; c++) value(t, c, v[c]);
#pragma unroll
                    for (int r = 0; r < RW; r++) {
                        const float w = sp[(row0 + r) * G_TOK + t];
                        if (!((line[r] >> t) & 1)) continue;
#pragma unroll
                        for (int c = 0; c < COLS; c++)
#pragma unroll
                            for (int e = 0; e < 4; e++) o[r][4 * c + e] = fmaf(w, v[c][e], o[r][4 * c + e]);
                    }
                }
            }
        }
        now = after;
    }
    if (!busy) return;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1)
#pragma unroll
        for (int r = 0; r < RW; r++) l[r] += __shfl_xor_sync(0xffffffffu, l[r], off);
#pragma unroll
    for (int r = 0; r < RW; r++) {
        if (row0 + r >= n_rows) continue;
        const int node = it.node0 + (row0 + r) / group, head = kvh * group + (row0 + r) % group;
        if (it.slot >= 0) {
            const int64_t at = (int64_t)(it.slot + node - it.node0) * H + head;
            if (lane == 0) p.part_ml[at] = make_float2(m[r], l[r]);
#pragma unroll
            for (int c = 0; c < COLS; c++) {
                const int e = 128 * c + 4 * lane;
                if (e < p.part_width) *reinterpret_cast<float4*>(p.part_o + at * p.part_width + e) = make_float4(o[r][4 * c], o[r][4 * c + 1], o[r][4 * c + 2], o[r][4 * c + 3]);
            }
        } else {
            const float M = p.sink ? fmaxf(m[r], 0.f) : m[r];
            const float w = exp2_approx(m[r] - M), total = l[r] * w + (p.sink ? exp2_approx(-M) : 0.f), scale = total == 0.f ? 0.f : w / total;
            T* out = static_cast<T*>(p.out) + ((int64_t)node * H + head) * dv;
#pragma unroll
            for (int c = 0; c < COLS; c++) {
                const int e = 128 * c + 4 * lane;
                if (dv % 4 == 0) {
                    if (e < dv) *reinterpret_cast<Pack<T, 4>*>(out + e) = {from_f32<T>(o[r][4 * c] * scale), from_f32<T>(o[r][4 * c + 1] * scale), from_f32<T>(o[r][4 * c + 2] * scale), from_f32<T>(o[r][4 * c + 3] * scale)};
                } else {
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        if (e + k < dv) out[e + k] = from_f32<T>(o[r][4 * c + k] * scale);
                }
            }
        }
    }
}

// The same for at most 16 rows (chains, small trees; fp32 of heads of 64 or 128: 8): eight warps share the rows' work instead of the rows.  A warp multiplies an eighth of the
// key's granules, the parts meet in shared memory, where every row has its warp for the softmax, and a warp has a quarter of the value's
// columns, a lane each, for half of the tile's tokens.  Bound by the chain of a tile.  (With a warp's rows its own, few rows leave most warps
// of a block idle and load one scheduler of the SM: one row of 2000 tokens, 32 fp32 heads of 128, 4 nodes 62 us instead of 24.)
template <typename T, int R, int COLS>  // COLS: columns of a lane
__global__ void __launch_bounds__(G_THREADS, 2) draft_few_kernel(const DraftParams p, const GenericSizes z) {
    extern __shared__ __align__(128) uint8_t raw[];
    __shared__ uint64_t bars[G_STAGES];
    constexpr int E = 16 / sizeof(T), MINE = (R + G_WARPS - 1) / G_WARPS;  // rows of a warp in the softmax
    float* const sq = reinterpret_cast<float*>(raw);     // [R][q_floats]
    float* const ss = sq + R * z.q_floats;               // [8][R][32] parts of scores; at the end [R][128 COLS], one half's output
    float* const sp = ss + G_WARPS * R * G_TOK;          // [R][32] weights
    float* const sa = sp + R * G_TOK;                    // [R] what the rows' earlier results are scaled by
    float2* const ml = reinterpret_cast<float2*>(sa + R);
    uint8_t* const stages = raw + whole((int)sizeof(float) * R * (z.q_floats + (G_WARPS + 1) * G_TOK + 3), 128);
    const int dk = p.d_key, dv = p.d_value;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = p.geo.n_heads, group = p.group, H = G * group;
    const int kvh = blockIdx.x % G;
    draft_lists_wait(p);
    const int4* const item = reinterpret_cast<const int4*>(p.items + blockIdx.x / G);
    const int4 ia = list_load(item), ib = list_load(item + 1), ic = list_load(item + 2);
    const DraftItem it = {ia.x, ia.y, ia.z, ia.w, ib.x, ib.y, ib.z, ib.w, {}};
    if (!draft_item_ok(p, ia, ib, R)) {
        if (tid == 0) atomicCAS(p.status, STATUS_OK, STATUS_BAD_WORK_LIST);
        return;
    }
    const int n_rows = it.n_nodes * group, k_gran = whole(dk, E) / E;
    Walk<T> tiles(p, z, it, kvh, stages, make_int2(ic.x, ic.y));
    Stages in = make_stages(p, bars);
    Tile now = tiles.take();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (now.n > 0) in.fetch(tiles, now, 0);
    if (warp < R) stage_queries<T, MINE>(p, it, kvh, sq, z.q_floats, n_rows, R, warp, G_WARPS);
    float m[MINE], l[MINE], o[R][COLS];
#pragma unroll
    for (int i = 0; i < MINE; i++) {
        m[i] = G_NEG_BIG;
        l[i] = 0.f;
    }
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int c = 0; c < COLS; c++) o[r][c] = 0.f;
    const int col0 = (warp & 3) * 32 * COLS + lane;  // and 32 further
    const int from_token = (warp >> 2) * (G_TOK / 2);
    // byte of column col0 + 32 c of token t: at[c] + t * v_line + the granule's place in the line, which goes by t & 7
    const int v_line = p.geo.v_swz ? 128 : z.v_bytes;
    int at[COLS], place[COLS];
#pragma unroll
    for (int c = 0; c < COLS; c++) {
        const int e = min(col0 + 32 * c, dv - 1), g = e / E;
        at[c] = G_TOK * z.k_bytes + e % E * (int)sizeof(T) + (p.geo.v_swz ? (g >> 3) * (G_TOK * 128) : g * 16);
        place[c] = g & 7;
    }
    const int swap = p.geo.v_swz ? 7 : 0;
    for (int stage = 0; now.n > 0; stage ^= 1) {
        if (!in.wait(stage)) return;  // nobody reads the tile before this one any more
        const Tile after = tiles.take();
        if (after.n > 0) in.fetch(tiles, after, stage ^ 1);
        const uint8_t* const sk = stages + stage * z.stage();
        auto value = [&](int t, int c) { return to_f32(*reinterpret_cast<const T*>(sk + at[c] + t * v_line + (swap ? (place[c] ^ (t & 7)) << 4 : 0))); };
        const bool drafted = now.chunk < 0;
        {
            float s[R];
#pragma unroll
            for (int r = 0; r < R; r++) s[r] = 0.f;
#pragma unroll 2
            for (int g = warp; g < k_gran; g += G_WARPS) {
                float k[E];
                Granule<T>::load(reinterpret_cast<const T*>(sk + staged(lane, g, z.k_bytes, p.geo.swz)), k);
#pragma unroll
                for (int r = 0; r < R; r++)
#pragma unroll
                    for (int e = 0; e < E; e += 4) {
                        const float4 q = *reinterpret_cast<const float4*>(sq + r * z.q_floats + g * E + e);
                        s[r] = fmaf(q.x, k[e], s[r]);
                        s[r] = fmaf(q.y, k[e + 1], s[r]);
                        s[r] = fmaf(q.z, k[e + 2], s[r]);
                        s[r] = fmaf(q.w, k[e + 3], s[r]);
                    }
            }
#pragma unroll
            for (int r = 0; r < R; r++) ss[(warp * R + r) * G_TOK + lane] = s[r];
        }
        const uint32_t there = now.n == 32 ? 0xffffffffu : (1u << now.n) - 1;
        __syncthreads();
        if (warp < R) {
            float s[MINE], high[MINE];
            bool see[MINE];
#pragma unroll
            for (int i = 0; i < MINE; i++) {
                const int r = min(warp + G_WARPS * i, R - 1);
                uint32_t line = there;
                if (drafted) line &= list_load(p.seen + (int64_t)(it.node0 + min(r, n_rows - 1) / group) * p.words + now.first / 32);
                see[i] = (line >> lane) & 1;
                float x = 0.f;
#pragma unroll
                for (int w = 0; w < G_WARPS; w++) x += ss[(w * R + r) * G_TOK + lane];
                s[i] = high[i] = see[i] ? x * p.scale_log2 : -INFINITY;
            }
#pragma unroll
            for (int off = 16; off >= 1; off >>= 1)
#pragma unroll
                for (int i = 0; i < MINE; i++) high[i] = fmaxf(high[i], __shfl_xor_sync(0xffffffffu, high[i], off));
#pragma unroll
            for (int i = 0; i < MINE; i++) {
                const int r = warp + G_WARPS * i;
                const float mn = fmaxf(m[i], high[i]), alpha = exp2_approx(m[i] - mn), w = see[i] ? exp2_approx(s[i] - mn) : 0.f;
                m[i] = mn;
                l[i] = l[i] * alpha + w;  // this lane's tokens only
                if (r < R) {
                    sp[r * G_TOK + lane] = w;
                    if (lane == 0) sa[r] = alpha;
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < R; r++) {
            const float alpha = sa[r];
#pragma unroll
            for (int c = 0; c < COLS; c++) o[r][c] *= alpha;
        }
        if (!drafted && now.n == G_TOK) {
#pragma unroll 2
            for (int t = 0; t < G_TOK / 2; t += 4) {
                float v[4][COLS];
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int c = 0; c < COLS; c++) v[i][c] = value(from_token + t + i, c);
#pragma unroll
                for (int r = 0; r < R; r++) {
                    const float4 w = *reinterpret_cast<const float4*>(sp + r * G_TOK + from_token + t);
#pragma unroll
                    for (int c = 0; c < COLS; c++) {
                        o[r][c] = fmaf(w.x, v[0][c], o[r][c]);
                        o[r][c] = fmaf(w.y, v[1][c], o[r][c]);
                        o[r][c] = fmaf(w.z, v[2][c], o[r][c]);
                        o[r][c] = fmaf(w.w, v[3][c], o[r][c]);
                    }
                }
            }
        } else {
            // values that a row does not see may be infinite: they are left out, not multiplied by zero
            uint32_t line[R];
            int node = it.node0, in_group = 0;
#pragma unroll
            for (int r = 0; r < R; r++) {
                line[r] = drafted && r < n_rows ? there & list_load(p.seen + (int64_t)node * p.words + now.first / 32) : there;
                if (++in_group == group) {
                    in_group = 0;
                    node++;
                }
            }
#pragma unroll 1
            for (int t = from_token; t < min(now.n, from_token + G_TOK / 2); t++) {
                float v[COLS];
#pragma unroll
                for (int c = 0; c < COLS; c++) v[c] = value(t, c);
#pragma unroll
                for (int r = 0; r < R; r++) {
                    const float w = sp[r * G_TOK + t];
#pragma unroll
                    for (int c = 0; c < COLS; c++) o[r][c] = (line[r] >> t) & 1 ? fmaf(w, v[c], o[r][c]) : o[r][c];
                }
            }
        }
        now = after;
    }
    if (warp < R) {
#pragma unroll
        for (int i = 0; i < MINE; i++) {
            const float sum = warp_sum(l[i]);
            if (lane == 0 && warp + G_WARPS * i < R) ml[warp + G_WARPS * i] = make_float2(m[i], sum);
        }
    }
    // the halves meet; the parts of scores have been read long ago
    if (warp >= 4) {
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int c = 0; c < COLS; c++) ss[r * 128 * COLS + col0 + 32 * c] = o[r][c];
    }
    __syncthreads();
    if (warp >= 4) return;
    int at_node = 0, in_group = 0;
#pragma unroll
    for (int r = 0; r < R; r++) {
        if (r >= n_rows) break;
        const int head = kvh * group + in_group;
        const float2 own = ml[r];
        const float M = p.sink && it.slot < 0 ? fmaxf(own.x, 0.f) : own.x;
        const float w = exp2_approx(own.x - M), total = own.y * w + (p.sink ? exp2_approx(-M) : 0.f), scale = total == 0.f ? 0.f : w / total;
        const int64_t row = (int64_t)((it.slot >= 0 ? it.slot : it.node0) + at_node) * H + head;
        if (it.slot >= 0 && tid == 0) p.part_ml[row] = own;
#pragma unroll
        for (int c = 0; c < COLS; c++) {
            const int e = col0 + 32 * c;
            const float x = o[r][c] + ss[r * 128 * COLS + e];
            if (it.slot >= 0) {
                if (e < p.part_width) p.part_o[row * p.part_width + e] = x;
            } else if (e < dv) {
                static_cast<T*>(p.out)[row * dv + e] = from_f32<T>(x * scale);
            }
        }
        if (++in_group == group) {
            in_group = 0;
            at_node++;
        }
    }
}

// fp32 with 9 rows and more, heads of 64 or 128: both products on the tensor cores (mma.sync, tf32), every operand as the sum of two tf32
// numbers of 11 bits and three products of the four, which leaves out 2^-22 of a product (fp32 products on the CUDA cores ran at 9 TFLOP/s).  Sums over
// more than four steps are fp32 additions, so that the error stays that of fp32 products: 5.1e-7 for 256 rows to a head over 16000 tokens (they have 6.4e-7).
// A block has 64 (32) rows; its warps are 4 (2) tiles of 16 rows times 2 (4) shares of every tile's 32 tokens, which meet at the end.  Up to 16 rows:
// eight shares of two tiles at a time, and no step of a tile waits for the other warps.
// S = Q K^T: m16n8k8, A = queries, B = keys.  O += P V: the weights stay where the scores were, if an MMA's k index 2 j + i is token 2 j + i for
// column j + 4 i: the values' rows are read in that order.
// Operands are split by whole-number instructions: by cvt.rna, of which an SM does few a cycle, 8 rows of 1000 tokens with 120 query rows to each of 8 heads of
// 64 took 98 us instead of 75.  One row of 4000 tokens, 32 heads of 128: 10 nodes 57 us, 8 nodes 57 (draft_few_kernel: 61 and 47); four rows of 288 and 9
// nodes 20 (29).  What bounds few rows now are instructions (1150 a warp and 64 tokens, a third of them waited for) and one block an SM.
struct Tf32Pair { uint32_t hi, lo; };
__device__ __forceinline__ Tf32Pair split_tf32(float x) {
    Tf32Pair r;
    // rounded up from half: what is not a number may wrap to zero here, and stays what it is in lo
    r.hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
    r.lo = __float_as_uint(x - __uint_as_float(r.hi)) & 0xffffe000u;
    return r;
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int D, int MT>  // head size; tiles of 16 rows
__global__ void __launch_bounds__(G_THREADS, MT == 1 && D == 128 ? 1 : 2) draft_tf32_kernel(const __grid_constant__ DraftParams p, const GenericSizes z) {
    extern __shared__ __align__(128) uint8_t raw[];
    constexpr int TILES = MT == 1 ? 2 : 1, STAGES = 2 * TILES;  // of 32 tokens, at a time
    constexpr bool SPLIT = MT == 1;                             // queries are staged as two numbers
    constexpr int SHARES = G_WARPS / MT, TILE_SHARES = SHARES / TILES, NT = G_TOK / TILE_SHARES / 8, ROWS = 16 * MT, QP = D + 4, OP = D + 4;
    __shared__ uint64_t bars[STAGES];
    float* const sq = reinterpret_cast<float*>(raw);     // [ROWS][QP], of pairs if SPLIT
    uint8_t* const stages = raw + whole((int)sizeof(float) * ROWS * QP * (SPLIT ? 2 : 1), 128);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quad = lane & 3, oct = lane >> 2;
    const int G = p.geo.n_heads, group = p.group, H = G * group;
    const int kvh = blockIdx.x % G;
    draft_lists_wait(p);
    const int4* const item = reinterpret_cast<const int4*>(p.items + blockIdx.x / G);
    const int4 ia = list_load(item), ib = list_load(item + 1), ic = list_load(item + 2);
    const DraftItem it = {ia.x, ia.y, ia.z, ia.w, ib.x, ib.y, ib.z, ib.w, {}};
    if (!draft_item_ok(p, ia, ib, ROWS)) {
        if (tid == 0) atomicCAS(p.status, STATUS_OK, STATUS_BAD_WORK_LIST);
        return;
    }
    const int n_rows = it.n_nodes * group, row0 = (warp % MT) * 16, mine = warp / MT / TILE_SHARES, tok0 = warp / MT % TILE_SHARES * (G_TOK / TILE_SHARES);
    const bool busy = row0 < n_rows;
    Walk<float> tiles(p, z, it, kvh, stages, make_int2(ic.x, ic.y));
    Stages in = make_stages(p, bars, STAGES);
    Tile now[TILES], after[TILES];
#pragma unroll
    for (int i = 0; i < TILES; i++) now[i] = tiles.take();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
#pragma unroll
    for (int i = 0; i < TILES; i++)
        if (now[i].n > 0) in.fetch(tiles, now[i], i);
    if constexpr (SPLIT) {
        float x[2][D / 32];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int r = min(warp + G_WARPS * i, n_rows - 1), at = r / group;
            const float* from = static_cast<const float*>(p.q) + (int64_t)(it.node0 + at) * p.q_node + (int64_t)(kvh * group + r - at * group) * p.q_head;
#pragma unroll
            for (int c = 0; c < D / 32; c++) x[i][c] = from[32 * c + lane];
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int c = 0; c < D / 32; c++) {
                const Tf32Pair a = split_tf32(x[i][c]);
                reinterpret_cast<uint2*>(sq)[(warp + G_WARPS * i) * QP + 32 * c + lane] = make_uint2(a.hi, a.lo);
            }
    } else {
#pragma unroll
        for (int half = 0; half < ROWS / G_WARPS; half += 4) stage_queries<float, 4>(p, it, kvh, sq, QP, n_rows, ROWS, warp * (ROWS / G_WARPS) + half, 1);
    }
    float o[D / 8][4], m[2] = {G_NEG_BIG, G_NEG_BIG}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < D / 8; i++)
#pragma unroll
        for (int k = 0; k < 4; k++) o[i][k] = 0.f;
    const uint32_t* line[2];  // of rows oct and oct + 8
#pragma unroll
    for (int h = 0; h < 2; h++) line[h] = p.seen + (int64_t)(it.node0 + min(row0 + oct + 8 * h, n_rows - 1) / group) * p.words;
    for (int stage = 0; now[0].n > 0; stage ^= TILES) {
        if (TILES == 2 && now[TILES - 1].n > 0) {
            if (!in.wait<TILES>(stage)) return;
        } else if (!in.wait(stage)) {
            return;
        }
        // nobody reads the tiles before these any more
#pragma unroll
        for (int i = 0; i < TILES; i++) {
            after[i] = tiles.take();
            if (after[i].n > 0) in.fetch(tiles, after[i], (stage ^ TILES) + i);
        }
        const Tile at = TILES == 2 && mine ? now[TILES - 1] : now[0];
        if (busy && tok0 < at.n) {
            const uint8_t* const sk = stages + (stage + mine) * z.stage();
            const uint8_t* const sv = sk + G_TOK * z.k_bytes;
            uint32_t see[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                see[h] = at.n == 32 ? 0xffffffffu : (1u << at.n) - 1;
                if (at.chunk < 0) see[h] &= list_load(line[h] + at.first / 32);
            }
            // Scores: products of the large parts in sums of four steps, which fp32 additions join (the tensor cores cut what they add, always towards zero);
            // those with a small part are 2^-11 of them and stay in their own.  Few rows: one tile of scores a warp, so twice as many sums of it, as
            // a chain of products is what takes time.
            constexpr int CHAINS = MT == 1 ? 2 : 1, STEPS = 4 * CHAINS;
            float s[NT][4], small[2 * CHAINS][NT][4];
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    s[n][k] = 0.f;
#pragma unroll
                    for (int c = 0; c < 2 * CHAINS; c++) small[c][n][k] = 0.f;
                }
#pragma unroll(MT == 1 || D == 64 ? 2 : 1)
            for (int k0 = 0; k0 < D / 8; k0 += STEPS) {
                float large[CHAINS][NT][4];
#pragma unroll
                for (int c = 0; c < CHAINS; c++)
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int k = 0; k < 4; k++) large[c][n][k] = 0.f;
#pragma unroll
                for (int j = 0; j < STEPS; j++) {
                    const int ks = k0 + j, c = j % CHAINS;
                    uint32_t ah[4], al[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const int e = (row0 + oct + 8 * (k & 1)) * QP + 8 * ks + quad + 4 * (k >> 1);
                        if constexpr (SPLIT) {
                            const uint2 a = reinterpret_cast<const uint2*>(sq)[e];
                            ah[k] = a.x;
                            al[k] = a.y;
                        } else {
                            const Tf32Pair a = split_tf32(sq[e]);
                            ah[k] = a.hi;
                            al[k] = a.lo;
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        const int t = tok0 + 8 * n + oct;
                        const float b0 = *reinterpret_cast<const float*>(sk + staged(t, 2 * ks, 0, 7) + 4 * quad), b1 = *reinterpret_cast<const float*>(sk + staged(t, 2 * ks + 1, 0, 7) + 4 * quad);
                        const Tf32Pair p0 = split_tf32(b0), p1 = split_tf32(b1);
                        mma_tf32(small[2 * c][n], al, p0.hi, p1.hi);
                        mma_tf32(small[2 * c + CHAINS - 1][n], ah, p0.lo, p1.lo);
                        mma_tf32(large[c][n], ah, p0.hi, p1.hi);
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int k = 0; k < 4; k++) s[n][k] += CHAINS == 2 ? large[0][n][k] + large[CHAINS - 1][n][k] : large[0][n][k];
            }
            float high[2] = {G_NEG_BIG, G_NEG_BIG};
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    s[n][k] += CHAINS == 2 ? (small[0][n][k] + small[1][n][k]) + (small[2 * CHAINS - 2][n][k] + small[2 * CHAINS - 1][n][k]) : small[0][n][k];
                    s[n][k] = (see[k >> 1] >> (tok0 + 8 * n + 2 * quad + (k & 1))) & 1 ? s[n][k] * p.scale_log2 : -INFINITY;
                    high[k >> 1] = fmaxf(high[k >> 1], s[n][k]);
                }
            float alpha[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                high[h] = fmaxf(high[h], __shfl_xor_sync(0xffffffffu, high[h], 1));
                high[h] = fmaxf(high[h], __shfl_xor_sync(0xffffffffu, high[h], 2));
                const float mn = fmaxf(m[h], high[h]);
                alpha[h] = exp2_approx(m[h] - mn);
                m[h] = mn;
                l[h] *= alpha[h];
            }
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    s[n][k] = exp2_approx(s[n][k] - m[k >> 1]);
                    l[k >> 1] += s[n][k];  // this lane's columns only: summed over the quad at the end
                }
            // The tile's part of the output in a sum of its own, small products first, which one fp32 operation adds: over the tokens of a long context the
            // cuts of one running sum would add up (64 rows of 16000 tokens: 4.4e-6 off)
            uint32_t ah[NT][4], al[NT][4];
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int k = 0; k < 4; k++) {  // A: row oct | oct + 8 of columns quad, then of quad + 4
                    const Tf32Pair a = split_tf32(s[n][2 * (k & 1) + (k >> 1)]);
                    ah[n][k] = a.hi;
                    al[n][k] = a.lo;
                }
#pragma unroll
            for (int i = 0; i < D / 8; i++) {
                const int c = 8 * i + oct;
                float part[4] = {0.f, 0.f, 0.f, 0.f};
                Tf32Pair b0[NT], b1[NT];
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    // values behind the tile's tokens are anything: zero
                    const int t = tok0 + 8 * n + 2 * quad;
                    const float v0 = *reinterpret_cast<const float*>(sv + staged(t, c >> 2, 0, 7) + 4 * (c & 3)), v1 = *reinterpret_cast<const float*>(sv + staged(t + 1, c >> 2, 0, 7) + 4 * (c & 3));
                    b0[n] = split_tf32(t < at.n ? v0 : 0.f);
                    b1[n] = split_tf32(t + 1 < at.n ? v1 : 0.f);
                    mma_tf32(part, al[n], b0[n].hi, b1[n].hi);
                    mma_tf32(part, ah[n], b0[n].lo, b1[n].lo);
                }
#pragma unroll
                for (int n = 0; n < NT; n++) mma_tf32(part, ah[n], b0[n].hi, b1[n].hi);
#pragma unroll
                for (int k = 0; k < 4; k++) o[i][k] = fmaf(o[i][k], alpha[k >> 1], part[k]);
            }
        }
#pragma unroll
        for (int i = 0; i < TILES; i++) now[i] = after[i];
    }
    // ---- the shares of a row meet
    __syncthreads();
    float* const so = reinterpret_cast<float*>(raw);                     // [8 warps][16][OP]
    float2* const ml = reinterpret_cast<float2*>(so + G_WARPS * 16 * OP);  // [8 warps][16]
#pragma unroll
    for (int h = 0; h < 2; h++) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        const int r = warp * 16 + oct + 8 * h;
        if (quad == 0) ml[r] = make_float2(m[h], l[h]);
#pragma unroll
        for (int i = 0; i < D / 8; i++) *reinterpret_cast<float2*>(so + r * OP + 8 * i + 2 * quad) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
    }
    __syncthreads();
    for (int r = warp; r < n_rows; r += G_WARPS) {
        const int at_node = r / group, head = kvh * group + r - at_node * group, from = (r / 16) * 16 + r % 16;
        float M = p.sink && it.slot < 0 ? 0.f : G_NEG_BIG, w[SHARES], total = 0.f;
#pragma unroll
        for (int k = 0; k < SHARES; k++) M = fmaxf(M, ml[from + k * 16 * MT].x);
#pragma unroll
        for (int k = 0; k < SHARES; k++) {
            const float2 part = ml[from + k * 16 * MT];
            w[k] = exp2_approx(part.x - M);
            total = fmaf(part.y, w[k], total);
        }
        float x[D / 32], bad = 0.f;
#pragma unroll
        for (int c = 0; c < D / 32; c++) {
            x[c] = 0.f;
#pragma unroll
            for (int k = 0; k < SHARES; k++) x[c] = fmaf(w[k], so[(from + k * 16 * MT) * OP + 32 * c + lane], x[c]);
            bad = fmaf(0.f, x[c], bad);
        }
        if (__any_sync(0xffffffffu, !(bad + 0.f * total == 0.f))) {
            // something infinite, perhaps where the row does not look: once more, a key at a time
            row_again<float>(p, it, kvh, r, lane);
            continue;
        }
        const int64_t row = (int64_t)((it.slot >= 0 ? it.slot : it.node0) + at_node) * H + head;
        if (it.slot >= 0) {
            if (lane == 0) p.part_ml[row] = make_float2(M, total);
#pragma unroll
            for (int c = 0; c < D / 32; c++) p.part_o[row * p.part_width + 32 * c + lane] = x[c];
        } else {
            if (p.sink) total += exp2_approx(-M);
            const float scale = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
            for (int c = 0; c < D / 32; c++) static_cast<float*>(p.out)[row * D + 32 * c + lane] = x[c] * scale;
        }
    }
}

constexpr int MOST_SHARED = 232448;  // of a CTA
bool tf32_serves(int block_rows, int dk, int dv, int esize) { return esize == 4 && block_rows > 8 && dk == dv && (dk == 64 || dk == 128); }

template <typename T>
cudaError_t launch_generic(const DraftParams& p, int block_rows, cudaStream_t stream) {
    const GenericSizes z = generic_sizes(p.d_key, p.d_value, sizeof(T));
    auto go = [&](auto* k, int threads, size_t floats) {
        const size_t smem = whole((int)(sizeof(float) * floats), 128) + (size_t)G_STAGES * z.stage();
        const cudaError_t e = allow_shared(reinterpret_cast<const void*>(k), MOST_SHARED - 128);  // less the barriers; other head sizes take other amounts
        if (e != cudaSuccess) return e;
        return launch_kernel(k, dim3((unsigned)p.n_items * p.geo.n_heads), threads, smem, 1, p.dependent & DEPENDENT_ATTENTION, stream, p, z);
    };
    auto few = [&](auto* k, int r) { return go(k, G_THREADS, (size_t)r * (z.q_floats + (G_WARPS + 1) * G_TOK + 3)); };
    auto many = [&](auto* k, int rw) { return go(k, G_THREADS, (size_t)G_WARPS * rw * (z.q_floats + G_TOK)); };
    if constexpr (sizeof(T) == 4) {
        if (tf32_serves(block_rows, p.d_key, p.d_value, 4) && p.geo.swz && p.geo.v_swz) {
            auto tf32 = [&](auto* k, int rows, int d) { return go(k, G_THREADS, std::max((size_t)rows * (d + 4), (size_t)G_WARPS * 16 * (d + 6) - G_STAGES * z.stage() / 4)); };
            const size_t few_floats = 2 * 16 * (p.d_key + 4) + 2 * z.stage() / 4;  // two stages more
            if (block_rows <= 16) return p.d_key == 64 ? go(&draft_tf32_kernel<64, 1>, G_THREADS, few_floats) : go(&draft_tf32_kernel<128, 1>, G_THREADS, few_floats);
            if (p.d_key == 64) return block_rows <= 32 ? tf32(&draft_tf32_kernel<64, 2>, 32, 64) : tf32(&draft_tf32_kernel<64, 4>, 64, 64);
            return block_rows <= 32 ? tf32(&draft_tf32_kernel<128, 2>, 32, 128) : tf32(&draft_tf32_kernel<128, 4>, 64, 128);
        }
    }
    if (p.d_value <= 128) {
        if (block_rows <= 4) return few(&draft_few_kernel<T, 4, 1>, 4);
        if (block_rows <= 8) return few(&draft_few_kernel<T, 8, 1>, 8);
        if (block_rows <= 12) return few(&draft_few_kernel<T, 12, 1>, 12);
        if (block_rows <= 16) return few(&draft_few_kernel<T, 16, 1>, 16);
        if (block_rows <= 32) return many(&draft_generic_kernel<T, 4, 1>, 4);
        return many(&draft_generic_kernel<T, 8, 1>, 8);
    }
    if (block_rows <= 4) return few(&draft_few_kernel<T, 4, 2>, 4);
    if (block_rows <= 8) return few(&draft_few_kernel<T, 8, 2>, 8);
    if (block_rows <= 12) return few(&draft_few_kernel<T, 12, 2>, 12);
    if (block_rows <= 16) return few(&draft_few_kernel<T, 16, 2>, 16);
    if (block_rows <= 32) return many(&draft_generic_kernel<T, 4, 2>, 4);
    return many(&draft_generic_kernel<T, 8, 2>, 8);
}

// ---- combination: a warp for every (node, query head) that several items serve ---------------------------------------------------
// Its latency is all there is to it: which partial results a node has is read while the kernel before still runs, where the work list has long been
// there, and their rows are requested together with the maxima and sums, eight at a time.
template <typename T, int COLS>
__global__ void __launch_bounds__(128) draft_merge_kernel(const DraftParams p) {
    constexpr int BATCH = COLS == 1 ? 8 : 4;
    const int H = p.geo.n_heads * p.group, lane = threadIdx.x & 31;
    const int pair = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (pair >= p.n_merge * H) return;
    draft_lists_wait(p);
    const int i = pair / H, head = pair % H;
    const int node = p.merge_nodes[i], b = p.merge_off[i], end = p.merge_off[i + 1];
    const bool there = (unsigned)node < (unsigned)p.n_nodes && b >= 0 && b <= end && end <= p.n_merge_slots;
    const int n = there ? end - b : 0;
    int slot = lane < n ? p.merge_slots[b + lane] : 0;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    auto bad = [&] {
        if (lane == 0) atomicCAS(p.status, STATUS_OK, STATUS_BAD_WORK_LIST);
    };
    if (!there) return bad();
    float M = p.sink ? 0.f : G_NEG_BIG, total = 0.f, o[COLS * 4];
#pragma unroll
    for (int c = 0; c < COLS * 4; c++) o[c] = 0.f;
    for (int s0 = 0; s0 < n; s0 += 32) {
        if (s0 > 0) slot = s0 + lane < n ? p.merge_slots[b + s0 + lane] : 0;
        if (__any_sync(0xffffffffu, (unsigned)slot >= (unsigned)p.n_slots)) return bad();
        const int here = min(32, n - s0);
        const int64_t at = (int64_t)slot * H + head;
        const float2 ml = lane < here ? p.part_ml[at] : make_float2(G_NEG_BIG, 0.f);
        float w = 0.f;
        for (int k0 = 0; k0 < here; k0 += BATCH) {
            float4 v[BATCH][COLS];
#pragma unroll
            for (int k = 0; k < BATCH; k++) {
                const int64_t from = __shfl_sync(0xffffffffu, at, min(k0 + k, here - 1)) * p.part_width;
#pragma unroll
                for (int c = 0; c < COLS; c++) {
                    const int e = 128 * c + 4 * lane;
                    v[k][c] = k0 + k < here && e < p.part_width ? *reinterpret_cast<const float4*>(p.part_o + from + e) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
            }
            if (k0 == 0) {
                const float high = fmaxf(M, warp_max(ml.x)), alpha = exp2f(M - high);
                M = high;
                w = exp2f(ml.x - M);
                total = total * alpha + ml.y * w;  // this lane's pieces
#pragma unroll
                for (int c = 0; c < COLS * 4; c++) o[c] *= alpha;
            }
#pragma unroll
            for (int k = 0; k < BATCH; k++) {
                const float wk = __shfl_sync(0xffffffffu, w, min(k0 + k, 31));
                if (k0 + k >= here) continue;
#pragma unroll
                for (int c = 0; c < COLS; c++) {
                    o[4 * c] = fmaf(wk, v[k][c].x, o[4 * c]);
                    o[4 * c + 1] = fmaf(wk, v[k][c].y, o[4 * c + 1]);
                    o[4 * c + 2] = fmaf(wk, v[k][c].z, o[4 * c + 2]);
                    o[4 * c + 3] = fmaf(wk, v[k][c].w, o[4 * c + 3]);
                }
            }
        }
    }
    total = warp_sum(total);
    if (p.sink) total += exp2f(-M);
    const float inv = total == 0.f ? 0.f : 1.f / total;
    T* out = static_cast<T*>(p.out) + ((int64_t)node * H + head) * p.d_value;
#pragma unroll
    for (int c = 0; c < COLS; c++) {
        const int e = 128 * c + 4 * lane;
        if (p.d_value % 4 == 0) {
            if (e < p.d_value) *reinterpret_cast<Pack<T, 4>*>(out + e) = {from_f32<T>(o[4 * c] * inv), from_f32<T>(o[4 * c + 1] * inv), from_f32<T>(o[4 * c + 2] * inv), from_f32<T>(o[4 * c + 3] * inv)};
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (e + k < p.d_value) out[e + k] = from_f32<T>(o[4 * c + k] * inv);
        }
    }
}

template <typename T>
cudaError_t merge(const DraftParams& p, cudaStream_t stream) {
    const int pairs = p.n_merge * p.geo.n_heads * p.group;
    const dim3 grid((unsigned)((pairs + 3) / 4));
    if (p.part_width <= 128) return launch_kernel(&draft_merge_kernel<T, 1>, grid, 128, 0, 1, p.dependent & DEPENDENT_MERGE, stream, p);
    return launch_kernel(&draft_merge_kernel<T, 2>, grid, 128, 0, 1, p.dependent & DEPENDENT_MERGE, stream, p);
}

// ---- acceptance: a warp per tree -------------------------------------------------------------------------------------------------
// A node is good when it is its parent's choice or probable enough; a line of good nodes from the first one down is accepted.  Whether
// a node's whole line is good is one look at the bits of the nodes that are not, so no walk from node to node is needed: latency
// is all there is to this kernel (2.5 us for a chain, 4.2 us for 256 trees of 63 nodes, of a call's 5.1).
__global__ void __launch_bounds__(32) accept_draft_kernel(const AcceptParams p) {
    __shared__ uint32_t bad[8];
    const int r = blockIdx.x, lane = threadIdx.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int first = p.first[r], n = p.first[r + 1] - first;
    for (int w = 0; w < p.words; w++) {
        const int i = 32 * w + lane;
        bool good = true;
        if (i < n) {
            const int parent = p.parent[first + i];
            if (parent >= 0) {
                good = p.tokens[first + i] == p.choice[first + parent];
                if (p.log_probs && !good) good = p.log_probs[first + i] >= fminf(p.log_epsilon, p.log_delta - p.entropy[first + parent]);
            }
        }
        const uint32_t b = __ballot_sync(0xffffffffu, !good);
        if (lane == 0) bad[w] = b;
    }
    __syncwarp();
    int best = -1;  // depth first, then the lower number
    for (int i = lane; i < n; i += 32) {
        bool whole = true;
        for (int w = 0; w < p.words; w++) whole = whole && (p.seen[(int64_t)(first + i) * p.words + w] & bad[w]) == 0;
        if (whole) best = max(best, p.depth[first + i] * 1024 + 1023 - i);
    }
    best = __reduce_max_sync(0xffffffffu, best);
    int count = 0;
    if (n > 0) {
        const int last = 1023 - (best & 1023);
        for (int w = 0; w < p.words; w++) {
            const uint32_t line = p.seen[(int64_t)(first + last) * p.words + w];
            if ((line >> lane) & 1) p.path[(int64_t)r * p.width + count + __popc(line & ((1u << lane) - 1))] = 32 * w + lane;
            count += __popc(line);
        }
        if (lane == 0) p.next[r] = p.choice[first + last];
    } else if (lane == 0) {
        p.next[r] = -1;
    }
    if (lane == 0) p.count[r] = count;
    for (int i = count + lane; i < p.width; i += 32) p.path[(int64_t)r * p.width + i] = -1;
}

}  // namespace

int draft_generic_ctas(int block_rows, int dk, int dv, int esize) {
    const GenericSizes z = generic_sizes(dk, dv, esize);
    if (block_rows <= 16 && tf32_serves(block_rows, dk, dv, esize)) return dk == 64 ? 2 * B200_SMS : B200_SMS;
    const int rows = sizeof(float) * block_rows * (z.q_floats + (block_rows <= 16 ? (G_WARPS + 1) * G_TOK + 3 : G_TOK));
    return B200_SMS * std::max(1, std::min(2, MOST_SHARED / (rows + G_STAGES * z.stage() + 1024 + 128)));
}

cudaError_t launch_draft_generic(const DraftParams& p, int block_rows, int dtype, cudaStream_t stream) {
    if (dtype == CA_DTYPE_F32) return launch_generic<float>(p, block_rows, stream);
    if (dtype == CA_DTYPE_F16) return launch_generic<__half>(p, block_rows, stream);
    return launch_generic<__nv_bfloat16>(p, block_rows, stream);
}

cudaError_t launch_draft_merge(const DraftParams& p, int dtype, cudaStream_t stream) {
    if (p.n_merge == 0) return cudaSuccess;
    if (dtype == CA_DTYPE_F32) return merge<float>(p, stream);
    if (dtype == CA_DTYPE_F16) return merge<__half>(p, stream);
    return merge<__nv_bfloat16>(p, stream);
}

cudaError_t launch_accept_draft(const AcceptParams& p, cudaStream_t stream) {
    return launch_kernel(&accept_draft_kernel, dim3(p.n_rows), 32, 0, 1, true, stream, p);
}

}  // namespace ca
