// Attention of drafted trees in any geometry and type (fp32 arithmetic on CUDA cores), the combination of partial results, and the
// walk that accepts drafted tokens.
//
// For node i of row r with query q, over the cached tokens C(r) of its row and its line A(i) (its ancestors and itself):
//   s_j = scale q . k_j,  m = max s_j,  l = sum e^(s_j - m),  out = sum e^(s_j - m) v_j / l,   j in C(r) u A(i)
// (sink: one more score of 0 without a value).  A piece of the keys yields (m, l, un-normalised out); pieces combine by
// out = sum 2^(m_p - M) O_p / sum 2^(m_p - M) l_p, with maxima in log2 units.
#include <algorithm>

#include "ca_draft.h"
#include "ca_kernels.h"
#include "ca_launch.cuh"
#include "ca_types.cuh"

namespace ca {
namespace {

constexpr int G_THREADS = 128, G_WARPS = 4, G_TOK = 32;
constexpr float G_NEG_BIG = -1.0e30f;

__host__ __device__ constexpr int round4(int x) { return (x + 3) & ~3; }
// floats between rows in shared memory: whole 16-byte granules, an odd number of them, so that 8 lanes reading a granule each of
// consecutive rows meet no bank twice
__host__ __device__ constexpr int pitch_of(int d) { return round4(d) + ((round4(d) / 4) % 2 == 0 ? 4 : 0); }

// One element of a stored tile as fp32
template <typename T> __device__ __forceinline__ float pool_elem(const T* tile, const Geometry& side, int t, int e) {
    return to_f32(tile[tile_elem_offset(side, t, e)]);
}

// An item for one key/value head.  Four warps with RW query rows each (row r: query head r % group of node r / group); the keys go by in tiles
// of 32 tokens, staged as fp32.  Scores: a lane has a token, and multiplies its key with the warp's rows (read by all lanes at once).
// Softmax: over the lanes.  Output: a lane has the columns 4 lane .. 4 lane + 3 of each 128, weights come from shared memory.
template <typename T, int RW, int COLS>  // COLS: groups of 128 value columns
__global__ void __launch_bounds__(G_THREADS) draft_generic_kernel(const DraftParams p) {
    extern __shared__ __align__(16) float smem[];
    const int dk = p.d_key, dv = p.d_value, kp = pitch_of(dk), vp = COLS * 128;
    float* const sq = smem;                              // [4 RW][kp]
    float* const sk = sq + G_WARPS * RW * kp;            // [32][kp]
    float* const sv = sk + G_TOK * kp;                   // [32][vp]
    float* const sp = sv + G_TOK * vp;                   // [4 RW][32] weights
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = p.geo.n_heads, group = p.group, H = G * group, C = p.geo.chunk_size;
    const int kvh = blockIdx.x % G;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int4 ia = __ldg(reinterpret_cast<const int4*>(p.items + blockIdx.x / G)), ib = __ldg(reinterpret_cast<const int4*>(p.items + blockIdx.x / G) + 1);
    const DraftItem it = {ia.x, ia.y, ia.z, ia.w, ib.x, ib.y, ib.z, ib.w, {}};
    if (!draft_item_ok(p, ia, ib, G_WARPS * RW)) {
        if (tid == 0) atomicCAS(p.status, STATUS_OK, STATUS_BAD_WORK_LIST);
        return;
    }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int n_rows = it.n_nodes * group;

    for (int i = tid; i < G_WARPS * RW * kp; i += G_THREADS) {
        const int r = i / kp, e = i % kp;
        float x = 0.f;
        if (r < n_rows && e < dk)
            x = to_f32(static_cast<const T*>(p.q)[(int64_t)(it.node0 + r / group) * p.q_node + (int64_t)(kvh * group + r % group) * p.q_head + e]);
        sq[i] = x;
    }
    float m[RW], l[RW], o[RW][COLS * 4];
#pragma unroll
    for (int r = 0; r < RW; r++) {
        m[r] = G_NEG_BIG;
        l[r] = 0.f;
#pragma unroll
        for (int c = 0; c < COLS * 4; c++) o[r][c] = 0.f;
    }
    const int row0 = warp * RW;
    const bool busy = row0 < n_rows;
    const Geometry k_side = tile_side(p.geo, 0), v_side = tile_side(p.geo, 1);

    // scores, softmax and output of the staged tile: n tokens, and for drafted ones which of them a row sees
    auto work = [&](int n, bool drafted, int word, int shift) {
        __syncthreads();
        if (busy) {
            float s[RW];
#pragma unroll
            for (int r = 0; r < RW; r++) s[r] = 0.f;
            for (int e = 0; e < dk; e += 4) {
                const float4 k = *reinterpret_cast<const float4*>(sk + lane * kp + e);
#pragma unroll
                for (int r = 0; r < RW; r++) {
                    const float4 q = *reinterpret_cast<const float4*>(sq + (row0 + r) * kp + e);
                    s[r] = fmaf(q.x, k.x, s[r]);
                    s[r] = fmaf(q.y, k.y, s[r]);
                    s[r] = fmaf(q.z, k.z, s[r]);
                    s[r] = fmaf(q.w, k.w, s[r]);
                }
            }
#pragma unroll
            for (int r = 0; r < RW; r++) {
                bool see = lane < n && row0 + r < n_rows;
                if (drafted && see) see = (p.seen[(int64_t)(it.node0 + (row0 + r) / group) * p.words + word] >> (shift + lane)) & 1;
                const float x = see ? s[r] * p.scale_log2 : -INFINITY;
                const float mn = fmaxf(m[r], warp_max(x));
                const float alpha = exp2f(m[r] - mn), w = see ? exp2f(x - mn) : 0.f;
                m[r] = mn;
                l[r] = l[r] * alpha + w;  // this lane's tokens only: summed over the lanes at the end
                sp[(row0 + r) * G_TOK + lane] = w;
                if (alpha != 1.f) {
#pragma unroll
                    for (int c = 0; c < COLS * 4; c++) o[r][c] *= alpha;
                }
            }
            __syncwarp();
            if (!drafted) {
#pragma unroll 1
                for (int t = 0; t < G_TOK; t += 4) {
                    float4 v[4][COLS];
#pragma unroll
                    for (int j = 0; j < 4; j++)
#pragma unroll
                        for (int c = 0; c < COLS; c++) v[j][c] = *reinterpret_cast<const float4*>(sv + (t + j) * vp + 128 * c + 4 * lane);
#pragma unroll
                    for (int r = 0; r < RW; r++) {
                        const float4 w4 = *reinterpret_cast<const float4*>(sp + (row0 + r) * G_TOK + t);
                        const float w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                        for (int j = 0; j < 4; j++)
#pragma unroll
                            for (int c = 0; c < COLS; c++) {
                                o[r][4 * c] = fmaf(w[j], v[j][c].x, o[r][4 * c]);
                                o[r][4 * c + 1] = fmaf(w[j], v[j][c].y, o[r][4 * c + 1]);
                                o[r][4 * c + 2] = fmaf(w[j], v[j][c].z, o[r][4 * c + 2]);
                                o[r][4 * c + 3] = fmaf(w[j], v[j][c].w, o[r][4 * c + 3]);
                            }
                    }
                }
            } else {
                // values of nodes that a row does not see may be infinite: they are left out, not multiplied by zero
#pragma unroll 1
                for (int t = 0; t < n; t++)
#pragma unroll
                    for (int r = 0; r < RW; r++) {
                        const bool see = row0 + r < n_rows && (p.seen[(int64_t)(it.node0 + (row0 + r) / group) * p.words + word] >> (shift + t)) & 1;
                        if (!see) continue;
                        const float w = sp[(row0 + r) * G_TOK + t];
#pragma unroll
                        for (int c = 0; c < COLS; c++) {
                            const float4 v = *reinterpret_cast<const float4*>(sv + t * vp + 128 * c + 4 * lane);
                            o[r][4 * c] = fmaf(w, v.x, o[r][4 * c]);
                            o[r][4 * c + 1] = fmaf(w, v.y, o[r][4 * c + 1]);
                            o[r][4 * c + 2] = fmaf(w, v.z, o[r][4 * c + 2]);
                            o[r][4 * c + 3] = fmaf(w, v.w, o[r][4 * c + 3]);
                        }
                    }
            }
        }
        __syncthreads();
    };

    for (int j = 0; j < it.n_tiles; j++) {
        int chunk = p.tiles[2 * (it.list + j)];
        const int in_chunk = p.tiles[2 * (it.list + j) + 1];
        if (chunk < 0 || chunk >= p.max_chunks || in_chunk > C) {
            if (tid == 0) atomicCAS(p.status, STATUS_OK, STATUS_BAD_WORK_LIST);
            continue;
        }
        const T* kt = static_cast<const T*>(p.pool) + tile_base_elems(p.geo, chunk, kvh, 0);
        const T* vt = kt + p.geo.tile_elems;
        for (int t0 = 0; t0 < in_chunk; t0 += G_TOK) {
            const int n = min(G_TOK, in_chunk - t0);
            constexpr int E = 16 / sizeof(T);
            if (p.geo.epg == E) {
                for (int i = tid; i < G_TOK * p.geo.gpr; i += G_THREADS) {
                    const int t = i / p.geo.gpr, g = i % p.geo.gpr;
                    float x[E];
#pragma unroll
                    for (int e = 0; e < E; e++) x[e] = 0.f;
                    if (t < n) Granule<T>::load(kt + tile_granule_index(p.geo, t0 + t, g) * E, x);
#pragma unroll
                    for (int e = 0; e < E; e += 4)
                        if (g * E + e < kp) *reinterpret_cast<float4*>(sk + t * kp + g * E + e) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
                }
                for (int i = tid; i < G_TOK * p.geo.v_gpr; i += G_THREADS) {
                    const int t = i / p.geo.v_gpr, g = i % p.geo.v_gpr;
                    float x[E];
#pragma unroll
                    for (int e = 0; e < E; e++) x[e] = 0.f;
                    if (t < n) Granule<T>::load(vt + tile_granule_index(v_side, t0 + t, g) * E, x);
#pragma unroll
                    for (int e = 0; e < E; e += 4) *reinterpret_cast<float4*>(sv + t * vp + g * E + e) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
                }
            } else {
                for (int i = tid; i < G_TOK * kp; i += G_THREADS) {
                    const int t = i / kp, e = i % kp;
                    sk[i] = t < n && e < dk ? pool_elem(kt, k_side, t0 + t, e) : 0.f;
                }
                for (int i = tid; i < G_TOK * dv; i += G_THREADS) {
                    const int t = i / dv, e = i % dv;
                    sv[t * vp + e] = t < n ? pool_elem(vt, v_side, t0 + t, e) : 0.f;
                }
            }
            work(n, false, 0, 0);
        }
    }
    for (int t0 = 0; t0 < it.n_drafted; t0 += G_TOK) {
        const int n = min(G_TOK, it.n_drafted - t0);
        for (int i = tid; i < G_TOK * kp; i += G_THREADS) {
            const int t = i / kp, e = i % kp;
            sk[i] = t < n && e < dk ? to_f32(static_cast<const T*>(p.k)[(int64_t)(it.tree + t0 + t) * p.k_node + (int64_t)kvh * p.k_head + e]) : 0.f;
        }
        for (int i = tid; i < G_TOK * dv; i += G_THREADS) {
            const int t = i / dv, e = i % dv;
            sv[t * vp + e] = t < n ? to_f32(static_cast<const T*>(p.v)[(int64_t)(it.tree + t0 + t) * p.v_node + (int64_t)kvh * p.v_head + e]) : 0.f;
        }
        work(n, true, t0 / 32, 0);
    }
    if (!busy) return;
#pragma unroll
    for (int r = 0; r < RW; r++) {
        const float sum = warp_sum(l[r]);
        if (row0 + r >= n_rows) continue;
        const int node = it.node0 + (row0 + r) / group, head = kvh * group + (row0 + r) % group;
        if (it.slot >= 0) {
            const int64_t at = (int64_t)(it.slot + node - it.node0) * H + head;
            if (lane == 0) p.part_ml[at] = make_float2(m[r], sum);
#pragma unroll
            for (int c = 0; c < COLS; c++) {
                const int e = 128 * c + 4 * lane;
                if (e < p.part_width) *reinterpret_cast<float4*>(p.part_o + at * p.part_width + e) = make_float4(o[r][4 * c], o[r][4 * c + 1], o[r][4 * c + 2], o[r][4 * c + 3]);
            }
        } else {
            const float M = p.sink ? fmaxf(m[r], 0.f) : m[r];
            const float w = exp2f(m[r] - M), total = sum * w + (p.sink ? exp2f(-M) : 0.f);
            T* out = static_cast<T*>(p.out) + ((int64_t)node * H + head) * dv;
#pragma unroll
            for (int c = 0; c < COLS; c++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int e = 128 * c + 4 * lane + k;
                    if (e < dv) out[e] = from_f32<T>(total == 0.f ? 0.f : o[r][4 * c + k] * w / total);
                }
        }
    }
}

template <typename T>
cudaError_t launch_generic(const DraftParams& p, int block_rows, cudaStream_t stream) {
    auto go = [&](auto* k, int rw, int cols) {
        const size_t smem = sizeof(float) * ((size_t)(G_WARPS * rw + G_TOK) * pitch_of(p.d_key) + G_TOK * cols * 128 + G_WARPS * rw * G_TOK);
        cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
        return launch_kernel(k, dim3((unsigned)p.n_items * p.geo.n_heads), G_THREADS, smem, 1, p.dependent & DEPENDENT_ATTENTION, stream, p);
    };
    if (p.geo.d_value <= 128 && p.d_value <= 128) {
        if (block_rows <= 16) return go(&draft_generic_kernel<T, 4, 1>, 4, 1);
        if (block_rows <= 32) return go(&draft_generic_kernel<T, 8, 1>, 8, 1);
        return go(&draft_generic_kernel<T, 16, 1>, 16, 1);
    }
    if (block_rows <= 16) return go(&draft_generic_kernel<T, 4, 2>, 4, 2);
    if (block_rows <= 32) return go(&draft_generic_kernel<T, 8, 2>, 8, 2);
    return go(&draft_generic_kernel<T, 16, 2>, 16, 2);
}

// ---- combination: a warp for every (node, query head) that several items serve ---------------------------------------------------
// Its latency is all there is to it: which partial results a node has is read while the kernel before still runs (the work list has long been
// there), and their rows are requested together with the maxima and sums, eight at a time.
template <typename T, int COLS>
__global__ void __launch_bounds__(128) draft_merge_kernel(const DraftParams p) {
    constexpr int BATCH = COLS == 1 ? 8 : 4;
    const int H = p.geo.n_heads * p.group, lane = threadIdx.x & 31;
    const int pair = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (pair >= p.n_merge * H) return;
    const int i = pair / H, head = pair % H;
    const int node = p.merge_nodes[i], b = p.merge_off[i], n = p.merge_off[i + 1] - b;
    int slot = lane < n ? p.merge_slots[b + lane] : 0;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    float M = p.sink ? 0.f : G_NEG_BIG, total = 0.f, o[COLS * 4];
#pragma unroll
    for (int c = 0; c < COLS * 4; c++) o[c] = 0.f;
    for (int s0 = 0; s0 < n; s0 += 32) {
        if (s0 > 0) slot = s0 + lane < n ? p.merge_slots[b + s0 + lane] : 0;
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
// is all there is to this kernel.
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
