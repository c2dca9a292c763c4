// Log probabilities, entropy and the best tokens of rows of logits, each logit read once.
//
//   M = max x,  l = sum 2^y,  a = sum y 2^y  with  y = (x - M) log2 e:
//   lse = M + ln l,   log p(t) = x_t - lse,   entropy = -sum p ln p = ln 2 (log2 l - a / l)
// held in fp32 relative to a running reference of each lane (moved when a logit exceeds it by more than 8 in log2 units), and combined over
// lanes, warps and CTAs by  l = sum 2^(m_i - M) l_i,  a = sum 2^(m_i - M) (a_i + (m_i - M) l_i).
//
// The best tokens: a warp keeps its best 32 in order, one a lane.  A vector of logits is looked at closer only when its largest reaches the
// threshold, the largest k-th best of any warp of the CTA; the first vectors give one to start with (k lanes whose maxima reach the k-th
// largest lane maximum hold k such logits).  Lists of two warps merge in six steps (bitonic).
#include <algorithm>
#include <cfloat>

#include "ca_kernels.h"
#include "ca_launch.cuh"
#include "ca_logits.h"
#include "ca_types.cuh"

namespace ca {
namespace {

constexpr int L_THREADS = 256, L_WARPS = L_THREADS / 32;
constexpr int L_UNROLL = 4;               // vectors of a lane that are requested together
constexpr float L_STEP = 8.f;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int NO_ID = 0x7fffffff;

// Excluded logits count as this finite value, so that 0 * y stays 0.  A power of two: its product with log2 e is exact, so a lane that has met
// nothing else gets y = 0 (rounded, the rest of 10^30 would be 10^22)
template <typename T> __device__ __forceinline__ constexpr float floor_of() { return -0x1p100f; }
template <> __device__ __forceinline__ constexpr float floor_of<__half>() { return -65504.f; }

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// a vector of logits as fp32
template <typename T> struct Vec {
    static constexpr int N = 16 / sizeof(T);
    uint4 raw;
    __device__ __forceinline__ void load(const T* p) {
        asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(raw.x), "=r"(raw.y), "=r"(raw.z), "=r"(raw.w) : "l"(p));
    }
    __device__ __forceinline__ void get(float (&x)[N]) const {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = __uint_as_float(w[i]);
        } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                x[2 * i] = __uint_as_float(w[i] << 16);
                x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                x[2 * i] = f.x;
                x[2 * i + 1] = f.y;
            }
        }
    }
};

struct Stat { float m, l, a; };  // reference (log2 units), sum, sum of y 2^y
__device__ __forceinline__ Stat join(Stat p, Stat q) {
    const float M = fmaxf(p.m, q.m), dp = p.m - M, dq = q.m - M, wp = exp2f(dp), wq = exp2f(dq);
    return {M, p.l * wp + q.l * wq, wp * (p.a + dp * p.l) + wq * (q.a + dq * q.l)};
}

struct Best { float v; int i; };
__device__ __forceinline__ bool better(float v, int i, float w, int j) { return v > w || (v == w && i < j); }
__device__ __forceinline__ Best shfl(Best b, int lane) { return {__shfl_sync(0xffffffffu, b.v, lane), __shfl_sync(0xffffffffu, b.i, lane)}; }
// two ordered lists, one entry a lane: the best 32 of both in order
__device__ __forceinline__ Best merge_lists(Best a, Best b, int lane) {
    b = shfl(b, 31 - lane);
    if (better(b.v, b.i, a.v, a.i)) a = b;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) {
        const Best o = {__shfl_xor_sync(0xffffffffu, a.v, off), __shfl_xor_sync(0xffffffffu, a.i, off)};
        if (better(o.v, o.i, a.v, a.i) == ((lane & off) == 0)) a = o;
    }
    return a;
}
__device__ __forceinline__ float sorted_down(float v, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int off = size >> 1; off >= 1; off >>= 1) {
            const float o = __shfl_xor_sync(0xffffffffu, v, off);
            const bool up = ((lane & off) == 0) == ((lane & size) == 0);  // this lane keeps the larger
            v = up ? fmaxf(v, o) : fminf(v, o);
        }
    return v;
}
// order-preserving whole numbers of floats, for atomicMax
__device__ __forceinline__ int ordered(float v) {
    const int b = __float_as_int(v);
    return b >= 0 ? b : b ^ 0x7fffffff;
}
__device__ __forceinline__ float from_ordered(int b) { return __int_as_float(b >= 0 ? b : b ^ 0x7fffffff); }

template <typename T, bool TOP> struct Walk {
    Stat st;
    Best best;
    int k, lane;
    int* shared_limit;

    __device__ __forceinline__ void insert(float v, int i) {
        const uint32_t worse = __ballot_sync(0xffffffffu, better(v, i, best.v, best.i));
        if (!worse) return;
        const int pos = __ffs(worse) - 1;
        const Best up = {__shfl_up_sync(0xffffffffu, best.v, 1), __shfl_up_sync(0xffffffffu, best.i, 1)};
        if (lane == pos) best = {v, i};
        if (lane > pos) best = up;
    }
    // x: logits of the ids from id on, which differ by lane, where `on`; floor: less than this is none of the best.  A whole warp
    template <int N> __device__ __forceinline__ void look(const float (&x)[N], int id, bool on, float floor) {
        const Best last = shfl(best, k - 1);
        uint32_t mine = 0;
#pragma unroll
        for (int e = 0; e < N; e++) {
            const float v = x[e] == x[e] ? x[e] : -INFINITY;
            if (on && v >= floor && better(v, id + e, last.v, last.i)) mine |= 1u << e;
        }
        if (!__any_sync(0xffffffffu, mine)) return;
#pragma unroll
        for (int e = 0; e < N; e++) {
            const float v = x[e] == x[e] ? x[e] : -INFINITY;
            uint32_t lanes = __ballot_sync(0xffffffffu, (mine >> e) & 1);
            while (lanes) {
                const int src = __ffs(lanes) - 1;
                lanes &= lanes - 1;
                insert(__shfl_sync(0xffffffffu, v, src), __shfl_sync(0xffffffffu, id, src) + e);
            }
        }
        const float kth = __shfl_sync(0xffffffffu, best.v, k - 1);
        if (lane == 0) atomicMax(shared_limit, ordered(kth));
    }
    template <int N> __device__ __forceinline__ void add(float (&x)[N], float high) {
        const float ref = high * LOG2E;
        if (!(ref <= st.m + L_STEP)) {
            const float d = st.m - ref, w = exp2f(d);
            st.a = w * (st.a + d * st.l);
            st.l *= w;
            st.m = ref;
        }
#pragma unroll
        for (int e = 0; e < N; e++) {
            const float y = fmaf(max_nan(x[e], floor_of<T>()), LOG2E, -st.m), w = exp2_approx(y);
            st.l += w;
            st.a = fmaf(w, y, st.a);
        }
    }
};

// A cluster of CTAs for every row; CTA 0 finishes it.
template <typename T, bool TOP>
__global__ void __launch_bounds__(L_THREADS) log_probs_kernel(const LogProbsParams p) {
    constexpr int N = Vec<T>::N;
    __shared__ Stat s_stat[L_WARPS];
    __shared__ Best s_best[L_WARPS][32];
    __shared__ int s_limit;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int S = p.splits, part = blockIdx.x % S, row = blockIdx.x / S;
    if (tid == 0) s_limit = ordered(-INFINITY);
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const T* x = static_cast<const T*>(p.logits) + (int64_t)row * p.row_stride;
    // vectors of the row, between a few logits before the first aligned address and behind the last
    const int head = min(p.vocab, (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)));
    const int n_vec = (p.vocab - head) / N, tail = p.vocab - head - n_vec * N;
    const int v0 = (int)((int64_t)n_vec * part / S), v1 = (int)((int64_t)n_vec * (part + 1) / S);

    Walk<T, TOP> w;
    w.st = {-3.0e38f, 0.f, 0.f};
    w.best = {-INFINITY, NO_ID};
    w.k = max(1, p.top);
    w.lane = lane;
    w.shared_limit = &s_limit;
    bool first = true;
    for (int b = v0; b < v1; b += L_THREADS * L_UNROLL) {
        Vec<T> v[L_UNROLL];
        bool on[L_UNROLL];
#pragma unroll
        for (int u = 0; u < L_UNROLL; u++) {
            const int i = b + u * L_THREADS + tid;
            on[u] = i < v1;
            if (on[u]) v[u].load(x + head + (int64_t)i * N);
        }
        float high[L_UNROLL];
#pragma unroll
        for (int u = 0; u < L_UNROLL; u++) {
            high[u] = -INFINITY;
            if (on[u]) {
                float f[N];
                v[u].get(f);
                high[u] = f[0];
#pragma unroll
                for (int e = 1; e < N; e++) high[u] = fmaxf(high[u], f[e]);
            }
        }
        if (TOP) {
            if (first) {
                float lane_high = high[0];
#pragma unroll
                for (int u = 1; u < L_UNROLL; u++) lane_high = fmaxf(lane_high, high[u]);
                const float sorted = sorted_down(lane_high == lane_high ? lane_high : -INFINITY, lane);
                if (lane == w.k - 1) atomicMax(&s_limit, ordered(sorted));
                first = false;
                __syncthreads();
            }
        }
#pragma unroll
        for (int u = 0; u < L_UNROLL; u++) {
            float f[N];
            v[u].get(f);
            if (TOP) {
                const float limit = from_ordered(*reinterpret_cast<volatile int*>(&s_limit));
                if (__any_sync(0xffffffffu, on[u] && !(high[u] < limit))) w.template look<N>(f, head + (b + u * L_THREADS + tid) * N, on[u], limit);
            }
            if (on[u]) w.add(f, fmaxf(high[u], floor_of<T>()));
        }
    }
    // the logits outside of whole vectors, one a lane
    if (warp == 0 && part == 0 && head > 0) {
        float f[1] = {lane < head ? to_f32(x[lane]) : -INFINITY};
        if (TOP) w.template look<1>(f, lane, lane < head, -INFINITY);
        if (lane < head) w.add(f, fmaxf(f[0], floor_of<T>()));
    }
    if (warp == L_WARPS - 1 && part == S - 1 && tail > 0) {
        const int at = p.vocab - tail + lane;
        float f[1] = {lane < tail ? to_f32(x[at]) : -INFINITY};
        if (TOP) w.template look<1>(f, at, lane < tail, -INFINITY);
        if (lane < tail) w.add(f, fmaxf(f[0], floor_of<T>()));
    }

    // ---- lanes, warps, CTAs
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1)
        w.st = join(w.st, {__shfl_xor_sync(0xffffffffu, w.st.m, off), __shfl_xor_sync(0xffffffffu, w.st.l, off), __shfl_xor_sync(0xffffffffu, w.st.a, off)});
    if (lane == 0) s_stat[warp] = w.st;
    if (TOP) s_best[warp][lane] = w.best;
#pragma unroll
    for (int half = L_WARPS / 2; half >= 1; half >>= 1) {
        __syncthreads();
        if (warp < half) {
            if (TOP) {
                w.best = merge_lists(w.best, s_best[warp + half][lane], lane);
                s_best[warp][lane] = w.best;
            }
            w.st = join(w.st, s_stat[warp + half]);
            if (lane == 0) s_stat[warp] = w.st;
        }
    }
    if (S > 1) {
        asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        if (part == 0 && warp == 0) {
            auto remote = [&](const void* here, int rank) {
                uint32_t a;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(here)), "r"(rank));
                return a;
            };
            auto read = [&](uint32_t a) {
                uint32_t v;
                asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
                return v;
            };
            for (int r = 1; r < S; r++) {
                const uint32_t a = remote(&s_stat[0], r);
                w.st = join(w.st, {__uint_as_float(read(a)), __uint_as_float(read(a + 4)), __uint_as_float(read(a + 8))});
                if (TOP) {
                    const uint32_t b = remote(&s_best[0][lane], r);
                    w.best = merge_lists(w.best, {__uint_as_float(read(b)), (int)read(b + 4)}, lane);
                }
            }
        }
        asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        if (part != 0) return;
    }
    if (warp != 0) return;
    // Nothing above the floor, or nothing that can be scaled: a row of lowest values (uniform over them), of nothing but excluded tokens, of
    // the largest values, of infinity.  Walked again as the formulas say.
    float log_l = logf(w.st.l), lse_m = w.st.m * LN2, entropy = log_l - LN2 * (w.st.a / w.st.l);
    if (w.st.m <= floor_of<T>() * LOG2E || w.st.m >= 1.0e37f) {
        float high = -INFINITY, sum = 0.f, weighted = 0.f;
        bool nan = false;
        for (int i = lane; i < p.vocab; i += 32) {
            const float f = to_f32(x[i]);
            nan = nan || f != f;
            high = fmaxf(high, f);
        }
        high = warp_max(high);
        for (int i = lane; i < p.vocab; i += 32) {
            const float d = to_f32(x[i]) - high, e = expf(d);  // infinity: not a number
            sum += e;
            if (e > 0.f) weighted = fmaf(e, d, weighted);
        }
        sum = warp_sum(sum);
        weighted = warp_sum(weighted);
        log_l = logf(sum);
        lse_m = high;
        entropy = log_l - weighted / sum;
        if (__any_sync(0xffffffffu, nan) || high == -INFINITY) log_l = lse_m = entropy = NAN;
    }
    if (lane == 0) {
        p.entropy[row] = entropy;
        p.lse[row] = make_float2(lse_m, log_l);
    }
    if (TOP && lane < p.top) {
        p.top_ids[(int64_t)row * p.top + lane] = w.best.i;
        p.top_log_probs[(int64_t)row * p.top + lane] = (w.best.v - lse_m) - log_l;
    }
}

template <typename T>
__global__ void __launch_bounds__(128) given_tokens_kernel(const LogProbsParams p) {
    const int i = blockIdx.x * 128 + threadIdx.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (i >= p.n_tokens) return;
    const int row = p.rows ? p.rows[i] : i, token = p.tokens[i];
    float lp = NAN;
    if (row >= 0 && row < p.n_rows) {
        const float2 lse = p.lse[row];
        if (token >= 0 && token < p.vocab) lp = (to_f32(static_cast<const T*>(p.logits)[(int64_t)row * p.row_stride + token]) - lse.x) - lse.y;
        if (token == -1) lp = 0.f;
    }
    p.log_probs[i] = lp;
}

template <typename T>
cudaError_t launch(const LogProbsParams& p, cudaStream_t stream) {
    if (p.n_rows > 0) {
        auto* k = p.top > 0 ? &log_probs_kernel<T, true> : &log_probs_kernel<T, false>;
        const cudaError_t e = launch_kernel(k, dim3((unsigned)(p.n_rows * p.splits)), L_THREADS, 0, p.splits, true, stream, p);
        if (e != cudaSuccess) return e;
    }
    if (p.n_tokens > 0) return launch_kernel(&given_tokens_kernel<T>, dim3((unsigned)((p.n_tokens + 127) / 128)), 128, 0, 1, true, stream, p);
    return cudaSuccess;
}

}  // namespace

// CTAs of a row: as many as fill the GPU a few times over, of at least 2048 logits each
int log_probs_splits(int n_rows, int vocab) {
    int s = 1;
    while (s < 8 && (int64_t)n_rows * s < 4 * B200_SMS && vocab / (2 * s) >= 2048) s *= 2;
    return s;
}

cudaError_t launch_log_probs(const LogProbsParams& p, int dtype, cudaStream_t stream) {
    if (dtype == CA_DTYPE_F32) return launch<float>(p, stream);
    if (dtype == CA_DTYPE_F16) return launch<__half>(p, stream);
    return launch<__nv_bfloat16>(p, stream);
}

}  // namespace ca
