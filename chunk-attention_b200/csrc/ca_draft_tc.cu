// Attention of drafted trees on the Blackwell tensor path: tcgen05.mma (fp16 or bf16) with accumulators in tensor memory.  For caches of
// 64-token chunks and head sizes of 64 or 128 elements, whose pool tiles are the tensor cores' own 128-byte-swizzled operand layout.
//
// A piece of work is (item, key/value head): up to 128 query rows (the query heads of a group for consecutive nodes; row r is head r % group of
// node r / group) against the item's chunks and, in the last piece of a row's private part, the drafted keys and values.
//   S = Q K^T      M = 128 rows, N = 64 tokens; D in TMEM, two buffers, so that S of tile j + 1 is computed under the softmax of tile j
//   softmax        one thread per row (= TMEM lane), fp32, log2 units; O is rescaled only when a row's maximum has grown by more than 8.
//                  The weights go back over S as hi + lo parts, whose sum has 16 bits of the fp32 weight (bf16; fp16: 22), so that what
//                  is left of rounding is that of the result
//   O += P V       A = P from TMEM, B = the V tile (MN-major panels)
// Pool tiles are bulk-copied verbatim; queries and drafted keys and values come by TMA tensor copies, which lay them out alike.  A drafted
// tile is masked by the bits of a row's line.  Rows leave as finished 16-bit rows where the item serves its nodes whole, else as
// fp32 partial results.
// Warp roles: 0-3 softmax and epilogue, 4 TMA producer over a ring of four tile slots, 5 TMEM and the MMA issue, 6 the next piece
// of work (a CTA takes over pieces that have not been launched yet: cluster launch control).  Two CTAs share an SM.
//
// What bounds it: with few rows to a tile HBM, and the ends of a piece (queries, first scores, last values, epilogue: 4.2 us together, of which
// the other CTA of the SM hides a part): 32 rows of 2048 shared and 512 own tokens, 32 heads, 13 nodes 84 us, 0.57 of the copy rate; 64 rows of up to 1024
// tokens, 8 heads of 4, 24 nodes 49 us (0.70).  With full blocks the tensor pipe, 384 cycles of scores (their operands' way from shared memory) and
// 512 of two products with V of some 1170 a tile: 8 rows of up to 16000, 8 heads of 8, 63 nodes 210 us.  One product with V would
// take 256 less, but rounds weights to 8 bits.
//
// A row of which an element comes out as not finite is computed once more on CUDA cores: a value that is infinite may be one that the row does
// not see (0 * infinity), and hi + lo parts of a weight times infinity are not its product.
//
// Every wait is bounded: on expiry a status code is recorded, every role falls through to the common exit, and the TMEM columns are
// freed there.
#include <cuda.h>

#include <atomic>

#include "ca_draft.h"
#include "ca_draft_row.cuh"
#include "ca_kernels.h"
#include "ca_launch.cuh"
#include "ca_ptx.cuh"
#include "ca_softmax.cuh"
#include "ca_tensor_map.h"
#include "ca_types.cuh"

namespace ca {
namespace {
using namespace ptx;

constexpr int A_ROWS = 128, A_TOK = 64, A_SLOTS = 4, A_THREADS = 256;
constexpr int A_SOFTMAX_REGS = 200, A_OTHER_REGS = 56;  // per thread; the block is launched with 2 x 128 (checked at the launch)
constexpr int A_TMEM_COLS = 256, A_COL_S = 128;
constexpr int A_NUM_BARS = 2 * A_SLOTS + 14;
constexpr float A_NEG_BIG = -1.0e30f, A_RESCALE_STEP = 8.f;

template <typename T> __host__ __device__ constexpr uint32_t idesc_of(int n, bool b_mn_major) {
    return umma_idesc_f16(A_ROWS, n, false, b_mn_major) | (std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u);
}
__device__ __forceinline__ void report(int* status, int code) { atomicCAS(status, STATUS_OK, code); }
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (std::is_same<T, __half>::value) {
        return pack_half2(lo, hi);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}
// 32 weights as pairs, and what their rounding left out
template <typename T> __device__ __forceinline__ void split_tile(const uint32_t (&s)[32], uint32_t* hi, uint32_t* lo) {
    if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float a = __uint_as_float(s[2 * i]), b = __uint_as_float(s[2 * i + 1]);
            hi[i] = pack_half2(a, b);
            const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi[i]));
            lo[i] = pack_half2(a - h.x, b - h.y);
        }
    } else {
        split_weights(s, hi, lo);
    }
}

// A piece of work as the roles read it; n_tiles = 0: there is none left
struct alignas(16) Work {
    int node0, n_rows, n_tiles, n_context;  // tiles in all, and from the pool
    int list, tree, n_drafted, slot;
    int n_nodes, kvh, pad[2];
    int2 head[4];  // the first tiles of the pool: slot, tokens
};

template <int DK, int DV> struct Sizes {
    static constexpr int Q_BYTES = A_ROWS * DK * 2, Q_PANEL = A_ROWS * 128;
    static constexpr int K_BYTES = A_TOK * DK * 2, V_BYTES = A_TOK * DV * 2;
    static constexpr int SLOT = K_BYTES > V_BYTES ? K_BYTES : V_BYTES;
    static constexpr int OUT_PITCH = 64 + 16;  // 64 bytes of a row at a time
    static constexpr int OUT = Q_BYTES + A_SLOTS * SLOT;
    static constexpr int WORK = OUT + A_ROWS * OUT_PITCH, CLC = WORK + 2 * (int)sizeof(Work), BARS = CLC + 16;
    static constexpr int SMEM = BARS + A_NUM_BARS * 8 + 8;
};

template <typename T, int DK, int DV>
__global__ void __launch_bounds__(A_THREADS, 2) draft_attn_kernel(const __grid_constant__ DraftParams p, const __grid_constant__ CUtensorMap q_map,
                                                                  const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
    using Z = Sizes<DK, DV>;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t sbase = smem_u32(smem);
    const uint32_t ring = sbase + Z::Q_BYTES;
    const uint32_t full_bar = sbase + Z::BARS;
    const uint32_t empty_bar = full_bar + 8 * A_SLOTS;
    const uint32_t s_full = empty_bar + 8 * A_SLOTS;  // [2]
    const uint32_t p_full = s_full + 16;              // [2]
    const uint32_t work_full = p_full + 16;           // [2]
    const uint32_t work_empty = work_full + 16;       // [2]
    const uint32_t o_done = work_empty + 16;
    const uint32_t o_free = o_done + 8;
    const uint32_t q_full = o_free + 8;
    const uint32_t q_empty = q_full + 8;
    const uint32_t clc_bar = q_empty + 8;
    const uint32_t ask_bar = clc_bar + 8;
    Work* const work = reinterpret_cast<Work*>(smem + Z::WORK);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Z::BARS + A_NUM_BARS * 8);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = p.geo.n_heads, group = p.group, H = G * group;
    // rows to nodes: r / group for r < 128 by a product (the quotient's fraction is 1 / group at least, the product is off by r / 65536 at most)
    const uint32_t by_group = (65536u + group - 1) / group;
    auto node_of = [&](int row) { return (int)((uint32_t)row * by_group >> 16); };

    if (threadIdx.x == 0) {
        for (int i = 0; i < A_SLOTS; i++) {
            mbar_init(full_bar + 8 * i, 1);
            mbar_init(empty_bar + 8 * i, 1);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(s_full + 8 * b, 1);
            mbar_init(p_full + 8 * b, 4 * 32);
            mbar_init(work_full + 8 * b, 1);
            mbar_init(work_empty + 8 * b, 4 * 32 + 2);
        }
        mbar_init(o_done, 1);
        mbar_init(o_free, 4 * 32);
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1);
        mbar_init(clc_bar, 1);
        mbar_init(ask_bar, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 5) {  // the warp that allocates is the warp that frees
        tmem_alloc(smem_u32(tmem_slot), A_TMEM_COLS);
        tmem_relinquish_alloc_permit();
    }
    tc_fence_before_thread_sync();
    __syncthreads();
    tc_fence_after_thread_sync();
    const uint32_t tmem_base = *tmem_slot;
    // with tensor memory in hand: a kernel behind this one may allocate, too.  Where the work list and the trees' bits have long been there (they came by
    // copies, which no kernel overtakes), only the producer waits for the kernels before: what is stored follows from what is loaded.
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    draft_lists_wait(p);
    // a wait of a single thread: false, with the code recorded, when the limit ran out
    auto wait = [&](uint32_t bar, int parity, int code) {
        if (mbar_wait_bounded(bar, parity, p.wait_limit)) return true;
        report(p.status, code);
        return false;
    };

    if (warp >= 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(A_OTHER_REGS));
        if (warp == 6 && lane == 0) {
            // ---- the next piece of work, asked for when the present one's last tiles are: a CTA that starts early, while the kernel before drains, must
            // not take what others will soon be there for (asked for at once, a wave of single pieces took twice its time back to back)
            int item = blockIdx.x;
            for (int n = 0;; n++) {
                if (n > 0) {
                    if (!wait(ask_bar, (n - 1) & 1, STATUS_EMPTY_WAIT_TIMEOUT) || !wait(work_empty + 8 * (n & 1), ((n >> 1) & 1) ^ 1, STATUS_EMPTY_WAIT_TIMEOUT)) break;
                    mbar_arrive_expect_tx(clc_bar, 16);
                    clc_try_cancel(sbase + Z::CLC, clc_bar);
                    if (!wait(clc_bar, (n - 1) & 1, STATUS_FULL_WAIT_TIMEOUT)) {
                        wait(clc_bar, (n - 1) & 1, STATUS_DRAIN_TIMEOUT);  // the answer is still on its way into this CTA's memory
                        break;
                    }
                    item = clc_block(sbase + Z::CLC);
                    fence_proxy_async();  // read before the next answer is written
                }
                Work w{};
                if (item >= 0) {
                    const int4* it = reinterpret_cast<const int4*>(p.items + item / G);
                    const int4 a = list_load(it), b = list_load(it + 1), c = list_load(it + 2), d = list_load(it + 3);
                    w.head[0] = make_int2(c.x, c.y);
                    w.head[1] = make_int2(c.z, c.w);
                    w.head[2] = make_int2(d.x, d.y);
                    w.head[3] = make_int2(d.z, d.w);
                    w.node0 = a.x;
                    w.n_nodes = a.y;
                    w.n_rows = a.y * group;
                    w.list = a.z;
                    w.n_context = a.w;
                    w.slot = b.x;
                    w.tree = b.y;
                    w.n_drafted = b.z;
                    w.n_tiles = a.w + (b.z + A_TOK - 1) / A_TOK;
                    w.kvh = item % G;
                    if (!draft_item_ok(p, a, b, A_ROWS)) {  // this CTA ends; pieces that have not been launched are others'
                        report(p.status, STATUS_BAD_WORK_LIST);
                        w.n_tiles = 0;
                        item = -1;
                    }
                }
                work[n & 1] = w;
                mbar_arrive(work_full + 8 * (n & 1));
                if (item < 0) break;
            }
        } else if (warp == 4 && lane == 0) {
            // ---- producer: slot i & 3 takes K of tile i / 2 (even i) or its V (odd i), i counted over all pieces
            int issued = 0, q_issued = 0, n = 0;
            asm volatile("griddepcontrol.wait;" ::: "memory");
            for (bool live = true; live; n++) {
                if (!wait(work_full + 8 * (n & 1), (n >> 1) & 1, STATUS_FULL_WAIT_TIMEOUT)) break;
                const Work w = work[n & 1];
                mbar_arrive(work_empty + 8 * (n & 1));
                if (w.n_tiles == 0) break;
                const int2* tiles = reinterpret_cast<const int2*>(p.tiles) + w.list;
                // asked for four tiles ahead: on its way while slots are waited for
                int2 queue[4] = {w.head[0], w.head[1], w.head[2], w.head[3]};
                for (int j = 0; j < w.n_tiles && live; j++) {
                    int2 tile = queue[0];
                    queue[0] = queue[1];
                    queue[1] = queue[2];
                    queue[2] = queue[3];
                    queue[3] = j + 4 < w.n_context ? list_load(tiles + j + 4) : make_int2(0, 0);
                    if (j < w.n_context && (tile.x < 0 || tile.x >= p.max_chunks || tile.y <= 0 || tile.y > A_TOK)) {
                        report(p.status, STATUS_BAD_WORK_LIST);  // keep the pipeline moving on a chunk that exists
                        tile = make_int2(0, A_TOK);
                    }
                    const uint8_t* src = static_cast<const uint8_t*>(p.pool) + ((size_t)tile.x * G + w.kvh) * (size_t)(Z::K_BYTES + Z::V_BYTES);
                    for (int side = 0; side < 2; side++) {
                        const int slot = issued & (A_SLOTS - 1);
                        if (!wait(empty_bar + 8 * slot, ((issued / A_SLOTS) & 1) ^ 1, STATUS_EMPTY_WAIT_TIMEOUT)) {
                            live = false;
                            break;
                        }
                        const uint32_t dst = ring + slot * Z::SLOT, bar = full_bar + 8 * slot;
                        const int panels = side ? DV / 64 : DK / 64;
                        if (j < w.n_context) {
                            const uint8_t* from = src + side * Z::K_BYTES;
                            mbar_arrive_expect_tx(bar, panels * tile.y * 128);
                            if (tile.y == A_TOK) {
                                bulk_copy_g2s(dst, from, panels * A_TOK * 128, bar);
                            } else {
                                for (int pn = 0; pn < panels; pn++) bulk_copy_g2s(dst + pn * (A_TOK * 128), from + pn * (A_TOK * 128), tile.y * 128, bar);
                            }
                        } else {
                            // lines past the drafted nodes are other trees' or zeros
                            mbar_arrive_expect_tx(bar, panels * A_TOK * 128);
                            for (int pn = 0; pn < panels; pn++)
                                tma_load_3d(dst + pn * (A_TOK * 128), side ? &v_map : &k_map, 64 * pn, w.kvh, w.tree + (j - w.n_context) * A_TOK, bar);
                        }
                        issued++;
                        if (side == 0 && j == max(0, w.n_tiles - 3)) mbar_arrive(ask_bar);
                        if (j == 0 && side == 0) {
                            // the queries follow the first K tile.  Rows past the block are other nodes' or zeros: nobody reads theirs
                            if (!wait(q_empty, (n & 1) ^ 1, STATUS_EMPTY_WAIT_TIMEOUT)) {
                                live = false;
                                break;
                            }
                            mbar_arrive_expect_tx(q_full, (DK / 64) * (A_ROWS / group) * group * 128);
#pragma unroll
                            for (int pn = 0; pn < DK / 64; pn++) tma_load_3d(sbase + pn * Z::Q_PANEL, &q_map, 64 * pn, w.kvh * group, w.node0, q_full);
                            q_issued++;
                        }
                    }
                }
            }
            for (int f = issued > A_SLOTS ? issued - A_SLOTS : 0; f < issued; f++)
                if (!wait(full_bar + 8 * (f & (A_SLOTS - 1)), (f / A_SLOTS) & 1, STATUS_DRAIN_TIMEOUT)) break;
            if (q_issued > 0) wait(q_full, (q_issued - 1) & 1, STATUS_DRAIN_TIMEOUT);  // pieces begun may be one more
        } else if (warp == 5 && elect_one()) {
            // ---- MMA issuer: one thread; t counts tiles over all pieces
            constexpr uint32_t DESC_HI = umma_desc_sw128_hi(1024);
            // a negative scale: the products of the negated queries (bit 13), so that the largest score stays the largest
            const uint32_t idesc_qk = idesc_of<T>(A_TOK, false) | (p.scale_log2 < 0.f ? 1u << 13 : 0u);
            constexpr uint32_t IDESC_PV = idesc_of<T>(DV, true);
            const uint32_t q_lo = umma_desc_sw128_lo(sbase, 16);
            auto issue_qk = [&](int t) {
                const int i = 2 * t, slot = i & (A_SLOTS - 1);
                if (!wait(full_bar + 8 * slot, (i / A_SLOTS) & 1, STATUS_FULL_WAIT_TIMEOUT)) return false;
                tc_fence_after_thread_sync();
                const uint32_t d = tmem_base + A_COL_S + (t & 1) * A_TOK;
                const uint32_t b_lo = umma_desc_sw128_lo(ring + slot * Z::SLOT, 16);
#pragma unroll
                for (int ks = 0; ks < DK / 16; ks++) {
                    const uint64_t a = umma_desc_pack(q_lo + (((ks >> 2) * Z::Q_PANEL + (ks & 3) * 32) >> 4), DESC_HI);
                    const uint64_t b = umma_desc_pack(b_lo + (((ks >> 2) * (A_TOK * 128) + (ks & 3) * 32) >> 4), DESC_HI);
                    umma_ss_f16(d, a, b, idesc_qk, ks > 0 ? 1u : 0u);
                }
                umma_commit(s_full + 8 * (t & 1));
                umma_commit(empty_bar + 8 * slot);
                return true;
            };
            int t = 0;
            bool live = true;
            for (int n = 0; live; n++) {
                if (!wait(work_full + 8 * (n & 1), (n >> 1) & 1, STATUS_FULL_WAIT_TIMEOUT)) break;
                const int n_tiles = work[n & 1].n_tiles;
                mbar_arrive(work_empty + 8 * (n & 1));
                if (n_tiles == 0) break;
                live = wait(q_full, n & 1, STATUS_FULL_WAIT_TIMEOUT) && issue_qk(t);
                if (live && n_tiles == 1) umma_commit(q_empty);
                for (int j = 0; j < n_tiles && live; j++, t++) {
                    if (j + 1 < n_tiles) {
                        if (!(live = issue_qk(t + 1))) break;
                        if (j + 2 == n_tiles) umma_commit(q_empty);
                    }
                    const int i = 2 * t + 1, slot = i & (A_SLOTS - 1);
                    live = wait(p_full + 8 * (t & 1), (t >> 1) & 1, STATUS_FULL_WAIT_TIMEOUT) &&
                           wait(full_bar + 8 * slot, (i / A_SLOTS) & 1, STATUS_FULL_WAIT_TIMEOUT) &&
                           (j > 0 || wait(o_free, (n & 1) ^ 1, STATUS_FULL_WAIT_TIMEOUT));  // the piece before has read its O
                    if (!live) break;
                    tc_fence_after_thread_sync();
                    const uint32_t a_tmem = tmem_base + A_COL_S + (t & 1) * A_TOK;  // hi parts, then lo parts, two per column
                    const uint32_t v_lo = umma_desc_sw128_lo(ring + slot * Z::SLOT, A_TOK * 128);
#pragma unroll
                    for (int part = 0; part < 2; part++)
#pragma unroll
                        for (int kk = 0; kk < 4; kk++) {
                            const uint64_t b = umma_desc_pack(v_lo + ((kk * 2048) >> 4), DESC_HI);
                            umma_ts_f16(tmem_base, a_tmem + part * 32 + kk * 8, b, IDESC_PV, (j > 0 || kk > 0 || part > 0) ? 1u : 0u);
                        }
                    umma_commit(empty_bar + 8 * slot);
                    umma_commit(o_done);
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(A_SOFTMAX_REGS));
        // ---- softmax: thread r owns query row r = TMEM lane r
        const int r = threadIdx.x;
        const float scale = fabsf(p.scale_log2);
        const uint32_t lane_addr = tmem_base + ((uint32_t)(warp * 32) << 16);
        uint8_t* const stage = smem + Z::OUT + warp * 32 * Z::OUT_PITCH;
        auto wait_all = [&](uint32_t bar, int parity) {  // by a whole warp
            const bool ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, p.wait_limit));
            if (!ok && lane == 0) report(p.status, STATUS_FULL_WAIT_TIMEOUT);
            return ok;
        };
        int t = 0;
        bool live = true;
        for (int n = 0; live; n++) {
            if (!wait_all(work_full + 8 * (n & 1), (n >> 1) & 1)) break;
            const Work w = work[n & 1];
            if (w.n_tiles == 0) break;
            const bool active = r < w.n_rows, busy = warp * 32 < w.n_rows;
            const int my_at = active ? node_of(r) : 0, my_node = w.node0 + my_at;
            const uint2* line = reinterpret_cast<const uint2*>(p.seen + (int64_t)my_node * p.words);
            float m_used = A_NEG_BIG, l = 0.f;
            for (int j = 0; j < w.n_tiles; j++, t++) {
                const int b = t & 1;
                const bool drafted = j >= w.n_context;
                const int stored = drafted ? 0 : (j == 0 ? w.head[0].y : list_load(p.tiles + 2 * (w.list + j) + 1));
                const int filled = drafted ? min(A_TOK, w.n_drafted - (j - w.n_context) * A_TOK) : max(0, min(A_TOK, stored));
                uint2 see = make_uint2(0u, 0u);
                if (drafted) see = list_load(line + (j - w.n_context));
                if (!(live = wait_all(s_full + 8 * b, (t >> 1) & 1))) break;
                tc_fence_after_thread_sync();
                float alpha = 1.f;
                bool rescale = false;
                if (busy) {
                    uint32_t s0[32], s1[32];
                    tmem_ld32(lane_addr + A_COL_S + b * A_TOK, s0);
                    tmem_ld32(lane_addr + A_COL_S + b * A_TOK + 32, s1);
                    tmem_wait_ld();
                    if (drafted || filled < A_TOK) {
                        if (!drafted) {
                            see.x = filled >= 32 ? 0xffffffffu : (1u << filled) - 1;
                            see.y = filled >= 64 ? 0xffffffffu : (filled > 32 ? (1u << (filled - 32)) - 1 : 0u);
                        }
#pragma unroll
                        for (int i = 0; i < 32; i++) {
                            if (!((see.x >> i) & 1)) s0[i] = 0xff800000u;
                            if (!((see.y >> i) & 1)) s1[i] = 0xff800000u;
                        }
                    }
                    const float mx = fmaxf(tile_max(s0, s1) * scale, A_NEG_BIG);
                    if (j == 0) {
                        m_used = mx;
                    } else if (mx > m_used + A_RESCALE_STEP) {
                        alpha = fast_exp2(m_used - mx);
                        m_used = mx;
                        l *= alpha;
                        rescale = true;
                    }
                    l += tile_weights(s0, s1, scale, m_used);
                    uint32_t pk[32], lo[32];
                    split_tile<T>(s0, pk, lo);
                    split_tile<T>(s1, pk + 16, lo + 16);
                    tmem_st32(lane_addr + A_COL_S + b * A_TOK, pk);
                    tmem_st32(lane_addr + A_COL_S + b * A_TOK + 32, lo);
                }
                // O += P V of tile t - 1 is complete (every thread follows o_done phase by phase)
                if (j > 0 && !(live = wait_all(o_done, (t - 1) & 1))) break;
                if (__any_sync(0xffffffffu, rescale)) {
                    tc_fence_after_thread_sync();
#pragma unroll 1
                    for (int c = 0; c < DV / 32; c++) {
                        uint32_t o[32];
                        tmem_ld32(lane_addr + c * 32, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                        tmem_st32(lane_addr + c * 32, o);
                    }
                }
                if (!drafted && filled < A_TOK) {
                    // The rows of V behind the tokens meet weights of zero, so they only have to be finite.  They are not copied: the slot's earlier
                    // tile, whose MMA of tile t - 2 is complete, may be another sequence's.  (A drafted tile's are other trees' or zeros.)
                    constexpr int PER_LINE = DV / 8;  // 16-byte granules of a row, 8 to a panel
                    const uint32_t to = ring + ((2 * t + 1) & (A_SLOTS - 1)) * Z::SLOT + ((r % PER_LINE) >> 3) * (A_TOK * 128) + (r & 7) * 16;
                    for (int t_line = filled + r / PER_LINE; t_line < A_TOK; t_line += 4 * 32 / PER_LINE) sts128_zero(to + t_line * 128);
                    fence_proxy_async();
                }
                tmem_wait_st();
                tc_fence_before_thread_sync();
                mbar_arrive(p_full + 8 * b);
            }
            if (!live || !(live = wait_all(o_done, (t - 1) & 1))) break;
            tc_fence_after_thread_sync();
            // ---- epilogue: rows are stored finished (16 bits) or partial (fp32).  Their sum shows whether an element is not finite.
            float scale_out = 1.f;
            uint64_t check = 0;
            const int64_t row_bytes = w.slot < 0 ? DV * 2 : p.part_width * 4;
            char* const base = (w.slot < 0 ? static_cast<char*>(p.out) : reinterpret_cast<char*>(p.part_o)) + (int64_t)(w.slot < 0 ? w.node0 : w.slot) * H * row_bytes;
            auto row_at = [&](int row) {
                const int at = node_of(row);
                return base + (int64_t)(at * H + w.kvh * group + row - at * group) * row_bytes;
            };
            if (w.slot < 0) {
                float total = l, M = m_used;
                if (p.sink) {
                    M = fmaxf(m_used, 0.f);
                    total = l * fast_exp2(m_used - M) + fast_exp2(-M);
                }
                scale_out = total == 0.f ? 0.f : fast_exp2(m_used - M) / total;
            } else if (active) {
                p.part_ml[(int64_t)(w.slot + my_at) * H + w.kvh * group + r - my_at * group] = make_float2(m_used, l);
            }
            // Up to 16 rows: a thread stores its own.  More: 32 columns (partial: 16) of a warp's rows at a time through shared memory, four lanes
            // to a row (128 rows straight from the threads: 15.6 us instead of 14.2 for one wave of pieces of two tiles; 13 rows through
            // shared memory: 9.7 instead of 9.0)
            const bool straight = w.n_rows <= 16;
            const int rows_here = min(32, w.n_rows - warp * 32);
            char* to[4];
#pragma unroll
            for (int k = 0; k < 4; k++) to[k] = straight ? (k == 0 ? row_at(r) : nullptr) : row_at(warp * 32 + 8 * k + (lane >> 2)) + 16 * (lane & 3);
            // A loop, not unrolled: this code runs once a piece, and straight through it the warps waited for instructions
#pragma unroll 1
            for (int c = 0; c < DV / 32; c++) {
                uint32_t o[32];
                if (busy) {
                    tmem_ld32(lane_addr + c * 32, o);
                    tmem_wait_ld();
                }
                if (c == DV / 32 - 1) {  // the accumulator may be overwritten
                    tc_fence_before_thread_sync();
                    mbar_arrive(o_free);
                }
                if (!busy) continue;
#pragma unroll
                for (int i = 0; i < 16; i++) check = add_f32x2(check, pair_u32(o[2 * i], o[2 * i + 1]));
                if (w.slot < 0) {
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        float a, bb;
                        unpair_f32(mul_f32x2(pair_u32(o[2 * i], o[2 * i + 1]), pair_f32(scale_out, scale_out)), a, bb);
                        o[i] = pack2<T>(a, bb);
                    }
                }
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    if (half == 1 && w.slot < 0) break;
                    const int at = w.slot < 0 ? 64 * c : 128 * c + 64 * half;
                    if (straight) {
                        if (active) {
#pragma unroll
                            for (int i = 0; i < 4; i++) *reinterpret_cast<uint4*>(to[0] + at + 16 * i) = make_uint4(o[16 * half + 4 * i], o[16 * half + 4 * i + 1], o[16 * half + 4 * i + 2], o[16 * half + 4 * i + 3]);
                        }
                        continue;
                    }
                    __syncwarp();  // what was staged before has been read
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        *reinterpret_cast<uint4*>(stage + lane * Z::OUT_PITCH + 16 * i) = make_uint4(o[16 * half + 4 * i], o[16 * half + 4 * i + 1], o[16 * half + 4 * i + 2], o[16 * half + 4 * i + 3]);
                    __syncwarp();
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const int rr = 8 * k + (lane >> 2);
                        const uint4 v = *reinterpret_cast<const uint4*>(stage + rr * Z::OUT_PITCH + 16 * (lane & 3));
                        if (rr < rows_here) *reinterpret_cast<uint4*>(to[k] + at) = v;
                    }
                }
            }
            __syncwarp();
            float sum_a, sum_b;
            unpair_f32(check, sum_a, sum_b);
            const uint32_t again = __ballot_sync(0xffffffffu, active && !(fabsf(sum_a) + fabsf(sum_b) + l < INFINITY));
            if (again) {
                __syncwarp();  // the rows above have been stored
                const DraftItem it = {w.node0, w.n_nodes, w.list, w.n_context, w.slot, w.tree, w.n_drafted, 0, {}};
                for (uint32_t rest = again; rest; rest &= rest - 1) row_again<T>(p, it, w.kvh, warp * 32 + __ffs(rest) - 1, lane);
            }
            mbar_arrive(work_empty + 8 * (n & 1));
        }
    }
    // ---- common exit: nobody touches TMEM after this barrier, then the allocating warp frees it
    tc_fence_before_thread_sync();
    __syncthreads();
    if (warp == 5) {
        tc_fence_after_thread_sync();
        tmem_dealloc(tmem_base, A_TMEM_COLS);
    }
}

// [nodes][heads][d] in boxes of one panel (64 elements) of some heads of some nodes
bool make_map(CUtensorMap* m, bool bf16, const void* base, int d, int64_t heads, int64_t nodes, int64_t head_stride, int64_t node_stride, int box_heads, int box_nodes) {
    const TensorMapEncode encode = tensor_map_encoder();
    if (!encode) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)heads, (cuuint64_t)nodes}, strides[2] = {(cuuint64_t)head_stride * 2, (cuuint64_t)node_stride * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_nodes}, step[3] = {1, 1, 1};
    return encode(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), dims, strides, box, step,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int DK, int DV>
cudaError_t launch(const DraftParams& p, cudaStream_t stream) {
    auto* k = draft_attn_kernel<T, DK, DV>;
    constexpr int smem = Sizes<DK, DV>::SMEM;
    static_assert(2 * (smem + 1024) <= 233472, "two CTAs do not fit in one SM's shared memory");
    constexpr bool bf16 = std::is_same<T, __nv_bfloat16>::value;
    const int G = p.geo.n_heads, H = G * p.group;
    CUtensorMap qm, km, vm;
    if (!make_map(&qm, bf16, p.q, DK, H, p.n_nodes, p.q_head, p.q_node, p.group, A_ROWS / p.group) ||
        !make_map(&km, bf16, p.k, DK, G, p.n_nodes, p.k_head, p.k_node, 1, A_TOK) || !make_map(&vm, bf16, p.v, DV, G, p.n_nodes, p.v_head, p.v_node, 1, A_TOK))
        return cudaErrorInvalidValue;
    // with fewer registers the warps would wait for them for good; what the compiler gave the kernel does not change
    static std::atomic<bool> ready;
    if (!ready) {
        cudaFuncAttributes have;
        cudaError_t e = cudaFuncGetAttributes(&have, k);
        if (e == cudaSuccess && 2 * have.numRegs < A_SOFTMAX_REGS + A_OTHER_REGS) e = cudaErrorInvalidConfiguration;
        if (e != cudaSuccess) return e;
        ready = true;
    }
    const cudaError_t e = allow_shared(reinterpret_cast<const void*>(k), smem);
    if (e != cudaSuccess) return e;
    return launch_kernel(k, dim3((unsigned)p.n_items * G), A_THREADS, smem, 1, p.dependent & DEPENDENT_ATTENTION, stream, p, qm, km, vm);
}

template <typename T>
cudaError_t launch_type(const DraftParams& p, cudaStream_t stream) {
    if (p.d_key == 128) return p.d_value == 128 ? launch<T, 128, 128>(p, stream) : launch<T, 128, 64>(p, stream);
    return p.d_value == 128 ? launch<T, 64, 128>(p, stream) : launch<T, 64, 64>(p, stream);
}

}  // namespace

bool draft_tc_serves(const Geometry& g, int d_key, int d_value, int group, float scale) {
    auto whole = [](int d) { return d == 64 || d == 128; };
    return g.esize == 2 && g.chunk_size == A_TOK && whole(d_key) && whole(d_value) && group <= A_ROWS && scale != 0.f;
}

cudaError_t launch_draft_tc(const DraftParams& p, int dtype, cudaStream_t stream) {
    return dtype == CA_DTYPE_F16 ? launch_type<__half>(p, stream) : launch_type<__nv_bfloat16>(p, stream);
}

}  // namespace ca
