// One row of an item of drafted attention by itself: for rows of which the tensor-core kernels give something that is not finite.
#pragma once
#include "ca_draft.h"
#include "ca_kernels.h"
#include "ca_types.cuh"

namespace ca {

// By a warp, a key at a time: lane e has the elements e, e + 32, e + 64, e + 96 (heads of up to 128).  What the row does not see is not read, and
// a weight meets its value in one product.
template <typename T>
__device__ __noinline__ void row_again(const DraftParams& p, const DraftItem& it, int kvh, int r, int lane) {
    const int G = p.geo.n_heads, group = p.group, H = G * group, dk = p.d_key, dv = p.d_value;
    const int node = it.node0 + r / group, head = kvh * group + r % group;
    const T* q = static_cast<const T*>(p.q) + (int64_t)node * p.q_node + (int64_t)head * p.q_head;
    float qe[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -1.0e30f, l = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) qe[i] = lane + 32 * i < dk ? to_f32(q[lane + 32 * i]) : 0.f;
    const Geometry vs = tile_side(p.geo, 1);
    auto take = [&](auto key, auto value) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (lane + 32 * i < dk) s = fmaf(qe[i], key(lane + 32 * i), s);
        s = warp_sum(s) * p.scale_log2;
        const float mn = fmaxf(m, s), alpha = exp2f(m - mn), x = exp2f(s - mn);
        m = mn;
        l = l * alpha + x;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (lane + 32 * i < dv) o[i] = o[i] * alpha + x * value(lane + 32 * i);
    };
    for (int j = 0; j < it.n_tiles; j++) {
        const int chunk = p.tiles[2 * (it.list + j)], n = min(p.tiles[2 * (it.list + j) + 1], p.geo.chunk_size);
        if (chunk < 0 || chunk >= p.max_chunks) continue;
        const T* kt = static_cast<const T*>(p.pool) + tile_base_elems(p.geo, chunk, kvh, 0);
        const T* vt = kt + p.geo.tile_elems;
        for (int t = 0; t < n; t++)
            take([&](int e) { return to_f32(kt[tile_elem_offset(p.geo, t, e)]); }, [&](int e) { return to_f32(vt[tile_elem_offset(vs, t, e)]); });
    }
    for (int t = 0; t < it.n_drafted; t++) {
        if (!((p.seen[(int64_t)node * p.words + t / 32] >> (t & 31)) & 1)) continue;
        const T* k = static_cast<const T*>(p.k) + (int64_t)(it.tree + t) * p.k_node + (int64_t)kvh * p.k_head;
        const T* v = static_cast<const T*>(p.v) + (int64_t)(it.tree + t) * p.v_node + (int64_t)kvh * p.v_head;
        take([&](int e) { return to_f32(k[e]); }, [&](int e) { return to_f32(v[e]); });
    }
    if (it.slot >= 0) {
        const int64_t at = (int64_t)(it.slot + node - it.node0) * H + head;
        if (lane == 0) p.part_ml[at] = make_float2(m, l);
        for (int i = 0; i < 4; i++)
            if (lane + 32 * i < dv) p.part_o[at * p.part_width + lane + 32 * i] = o[i];
    } else {
        const float M = p.sink ? fmaxf(m, 0.f) : m, x = exp2f(m - M), total = l * x + (p.sink ? exp2f(-M) : 0.f);
        for (int i = 0; i < 4; i++)
            if (lane + 32 * i < dv) static_cast<T*>(p.out)[((int64_t)node * H + head) * dv + lane + 32 * i] = from_f32<T>(total == 0.f ? 0.f : o[i] * x / total);
    }
}

}  // namespace ca
