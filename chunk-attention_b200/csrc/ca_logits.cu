// Log probabilities, entropy and the best tokens of rows of logits, each logit read once.
//
//   M = max x,  l = sum 2^y,  a = sum y 2^y  with  y = (x - M) log2 e:
//   lse = M + ln l,   log p(t) = x_t - lse,   entropy = -sum p ln p = ln 2 (log2 l - a / l)
// held in fp32 relative to a running reference of each lane (moved when a logit exceeds it by more than 8 in log2 units), and combined over
// lanes, warps and CTAs by  l = sum 2^(m_i - M) l_i,  a = sum 2^(m_i - M) (a_i + (m_i - M) l_i).
//
// The best tokens: groups of threads know their largest logit, and the k-th largest of these is a threshold that k logits reach and hardly more do.
// It is taken from the first vectors and again after 4, 16 ... times as many; vectors with a logit that reaches it are noted (some k
// each time).  At the end those logits of them that reach the last threshold are put in order.  Rows of which that finds too few (excluded tokens)
// or too many (rising or equal logits) go by insertion.
//
// What bounds it: instructions (an exponential and some five others a logit) at 0.6 to 0.75 of the copy rate, then the second kernel's chain of
// dependent reads.  2048 rows of 128000 in bf16 with 20 best 128 us (floor 80), 1536 rows of 32000 in fp16 with one 34 (15), 517 rows of 50001 in fp32
// with 8 30 (16); one row of 32000 in fp32 with 5 by a cluster 7.5 us.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "../../include/chunk_attn_b200.h"
#include "ca_kernels.h"
#include "ca_launch.cuh"
#include "ca_ptx.cuh"
#include "ca_logits.h"
#include "ca_types.cuh"

namespace ca {

__device__ int g_log_probs_status = 0;

namespace {

// Eight vectors a thread and turn: a turn's own work (waits, the threshold) is some 80 instructions, a vector's about 40.  Four a turn in blocks of 256
// threads, which leave half of the registers: 85 instructions a vector with one best token, 144 us for 2048 rows of 128000 in bf16.
constexpr int L_THREADS = 128, L_WARPS = L_THREADS / 32;
constexpr int L_UNROLL = 8;               // vectors that a thread takes in a turn
constexpr int L_STEP = L_THREADS * L_UNROLL;
constexpr int L_STAGES = 3;
constexpr int L_RING = L_STAGES * L_STEP * 16;
constexpr long long L_WAIT_LIMIT = DEFAULT_WAIT_LIMIT_CYCLES;
constexpr int L_HITS = LOG_PROBS_HITS;    // threads' turns of which a logit reached the threshold of its time
constexpr int L_FOUND = 256;              // logits that reach the last one
constexpr int L_GROUPS = 64;              // of threads, at most
constexpr int L_ROWS = 3;                 // rows that may be at hand: one is begun, one finished, one cleared
constexpr int F_THREADS = 128, F_WARPS = F_THREADS / 32;
constexpr float L_RESCALE = 8.f;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float L_HIGHEST = 0x1p30f;      // references from here on leave more of their rounding in the exponents than 2^y can hold
constexpr int NO_ID = 0x7fffffff;

// Excluded and masked logits count as this finite value at least, so that 0 * y stays 0.  A reference is a rounded product, high * log2 e, and what its
// rounding leaves stands in the exponents of the lane: half a step of the product, 64 at 2^30, which 2^y can hold (next to -10^10 512, which
// it cannot: a lane that had met nothing but such masks made its whole row NaN).  A logit above the floor is above it by 64 (fp32) at least, so e^-64
// of it is all that a lower one may count too much.
template <typename T> __device__ __forceinline__ constexpr float floor_of() { return -0x1p30f; }
template <> __device__ __forceinline__ constexpr float floor_of<__half>() { return -65504.f; }
// The least threshold: the bf16 (fp16) number above it
template <typename T> __device__ __forceinline__ constexpr float least_of() { return -0x1.fep29f; }
template <> __device__ __forceinline__ constexpr float least_of<__half>() { return -65472.f; }

// A vector of logits, 16 bytes
template <typename T> struct Vec {
    static constexpr int N = 16 / sizeof(T);
    uint32_t w[4];
    __device__ __forceinline__ void load(const T* p) {
        asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(p));
    }
    __device__ __forceinline__ void load_shared(uint32_t a) {
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(a));
    }
    __device__ __forceinline__ void get(float (&x)[N]) const {
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
    // lifts everything to floor_of() (what is not a number stays so); the largest that are numbers, of a 16-bit type still one of each half
    __device__ __forceinline__ uint32_t lift() {
        uint32_t a, b;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; i++) asm("max.NaN.f32 %0, %0, %1;" : "+f"(reinterpret_cast<float&>(w[i])) : "f"(floor_of<T>()));
            return __float_as_uint(fmaxf(fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1])), fmaxf(__uint_as_float(w[2]), __uint_as_float(w[3]))));
        } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
            for (int i = 0; i < 4; i++) asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(w[i]) : "r"(0xce80ce80u));
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(w[i]) : "r"(0xfbfffbffu));
        }
        a = larger(w[0], w[1]);
        b = larger(w[2], w[3]);
        return larger(a, b);
    }
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
        uint32_t r;
        if constexpr (sizeof(T) == 4) r = __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
        else if constexpr (std::is_same<T, __nv_bfloat16>::value) asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        else asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ float value(uint32_t a) {
        if constexpr (sizeof(T) == 4) return __uint_as_float(a);
        else if constexpr (std::is_same<T, __nv_bfloat16>::value) return fmaxf(__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u));
        else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&a));
            return fmaxf(f.x, f.y);
        }
    }
    static constexpr uint32_t NOTHING = sizeof(T) == 4 ? 0xff800000u : (std::is_same<T, __nv_bfloat16>::value ? 0xff80ff80u : 0xfc00fc00u);  // -infinity
};

struct Stat { float m, l, a; };  // reference (log2 units), sum, sum of y 2^y
__device__ __forceinline__ Stat join(Stat p, Stat q) {
    const float M = fmaxf(p.m, q.m), dp = p.m - M, dq = q.m - M, wp = exp2_approx(dp), wq = exp2_approx(dq);
    return {M, p.l * wp + q.l * wq, wp * (p.a + dp * p.l) + wq * (q.a + dq * q.l)};
}
// The running sums of a lane, in pairs
struct Sums {
    float m = -3.0e38f;
    uint64_t l = 0, a = 0;
    __device__ __forceinline__ void move(float high) {  // the reference, where the largest to come is far above it
        const float ref = high * LOG2E;
        if (!(ref <= m + L_RESCALE)) {
            const float d = m - ref, w = exp2_approx(d);
            const uint64_t w2 = pair_f32(w, w);
            a = mul_f32x2(w2, fma_f32x2(pair_f32(d, d), l, a));
            l = mul_f32x2(w2, l);
            m = ref;
        }
    }
    template <int N> __device__ __forceinline__ void add(const float (&x)[N]) {  // N even
        const uint64_t log2e = pair_f32(LOG2E, LOG2E), minus = pair_f32(-m, -m);
#pragma unroll
        for (int e = 0; e < N; e += 2) {
            const uint64_t y = fma_f32x2(pair_f32(x[e], x[e + 1]), log2e, minus);
            float y0, y1;
            unpair_f32(y, y0, y1);
            const uint64_t w = pair_f32(exp2_approx(y0), exp2_approx(y1));
            l = add_f32x2(l, w);
            a = fma_f32x2(w, y, a);
        }
    }
    __device__ __forceinline__ void add_one(float x, float floor) {
        float t;
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(t) : "f"(x), "f"(floor));
        const float ref = fmaxf(t, floor) * LOG2E;
        const float M = fmaxf(m, ref), y = fmaf(t, LOG2E, -M), w = exp2_approx(y);
        Stat s = total(), one = {M, w, w * y};
        s = join(s, one);
        m = s.m;
        l = pair_f32(s.l, 0.f);
        a = pair_f32(s.a, 0.f);
    }
    __device__ __forceinline__ Stat total() const {
        float l0, l1, a0, a1;
        unpair_f32(l, l0, l1);
        unpair_f32(a, a0, a1);
        return {m, l0 + l1, a0 + a1};
    }
};

struct Best { float v; int i; };
__device__ __forceinline__ bool better(Best a, Best b) { return a.v > b.v || (a.v == b.v && a.i < b.i); }
__device__ __forceinline__ Best shfl(Best b, int lane) { return {__shfl_sync(0xffffffffu, b.v, lane), __shfl_sync(0xffffffffu, b.i, lane)}; }
__device__ __forceinline__ Best shfl_xor(Best b, int off) { return {__shfl_xor_sync(0xffffffffu, b.v, off), __shfl_xor_sync(0xffffffffu, b.i, off)}; }
// two ordered lists, one entry a lane: the best 32 of both in order
__device__ __forceinline__ Best merge_lists(Best a, Best b, int lane) {
    b = shfl(b, 31 - lane);
    if (better(b, a)) a = b;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) {
        const Best o = shfl_xor(a, off);
        if (better(o, a) == ((lane & off) == 0)) a = o;
    }
    return a;
}
// order-preserving whole numbers of floats
__device__ __forceinline__ int ordered(float v) {
    const int b = __float_as_int(v);
    return b >= 0 ? b : b ^ 0x7fffffff;
}
__device__ __forceinline__ float from_ordered(int b) { return __int_as_float(b >= 0 ? b : b ^ 0x7fffffff); }

struct Shared {
    uint64_t full[L_STAGES], empty[L_STAGES];
    float group[L_ROWS][L_GROUPS];
    Stat stat[L_ROWS][L_WARPS];
    int n_hits[L_ROWS];
    int n_found;
    float limit;
    double2 lse;
    union {
        uint32_t hits[L_ROWS][L_HITS];
        struct {                    // a row that a cluster finishes is the only one
            uint32_t own[L_HITS];
            Best found[L_FOUND];
            Best list[L_WARPS][32]; // [0]: the best, in order; of the slow way: each warp's
        } one;
    };
};

// k-th largest of the groups' largest logits, as far as they are known: every one of them is a logit of its group, so k logits reach it.  Others may
// be telling theirs: all lanes go by what they have read once.  Up to 24 best tokens by 32 groups of 4 threads (24: some 44 logits reach the
// threshold), else by 64 of 2, which takes three times as long.
__device__ __forceinline__ bool wide_groups(int k) { return k <= 24; }
__device__ __forceinline__ float kth_of_groups(const volatile float* group, int k, int lane) {
    const float v = group[lane];
    int above_v = 0, least = ordered(INFINITY);
    if (wide_groups(k)) {
#pragma unroll
        for (int i = 0; i < 32; i++) above_v += __shfl_sync(0xffffffffu, v, i) > v;
    } else {
        const float w = group[32 + lane];
        int above_w = 0;
#pragma unroll
        for (int i = 0; i < 32; i++) {
            const float a = __shfl_sync(0xffffffffu, v, i), b = __shfl_sync(0xffffffffu, w, i);
            above_v += (a > v) + (b > v);
            above_w += (a > w) + (b > w);
        }
        if (above_w < k) least = ordered(w);
    }
    if (above_v < k) least = min(least, ordered(v));
    return from_ordered(__reduce_min_sync(0xffffffffu, least));
}
// A note of a thread's turn: the turn of its stretch, the thread, a bit for every vector of which a logit reached the threshold
static_assert(L_THREADS == 128 && L_UNROLL == 8, "a note has 7 bits for the thread, 8 for its vectors and 17 for the turn");
__device__ __forceinline__ uint32_t note_of(int turn, int thread, uint32_t vectors) { return (uint32_t)turn << 15 | (uint32_t)thread << 8 | vectors; }
// The logits of noted vectors that reach the threshold; v0: the stretch's first vector
template <typename T, typename F> __device__ __forceinline__ void look_at(const T* body, int first_id, int v0, const uint32_t* notes, int n, float limit, int start, int step, F keep) {
    constexpr int N = Vec<T>::N;
    for (int h = start; h < n; h += step) {
        const uint32_t note = notes[h];
        for (uint32_t rest = note & 255; rest; rest &= rest - 1) {
            const int at = v0 + (int)(note >> 15) * L_STEP + (__ffs(rest) - 1) * L_THREADS + (int)((note >> 8) & 127);
            Vec<T> v;
            v.load(body + (int64_t)at * N);
            float f[N];
            v.get(f);
#pragma unroll
            for (int e = 0; e < N; e++)
                if (f[e] >= limit) keep(f[e], first_id + at * N + e);
        }
    }
}
// A logit's place is how many are better
__device__ __forceinline__ void put_in_order(const Best* found, int n, Best* list, int start, int step) {
    for (int i = start; i < n; i += step) {
        const Best me = found[i];
        int place = 0;
        for (int j = 0; j < n; j++) place += better(found[j], me);
        if (place < 32) list[place] = me;
    }
}

// The best of logits [lo, hi) by insertion into ordered lists, whatever they are: for rows of which the threshold found too few (excluded tokens)
// or too many (rising or equal logits).  Returns this warp's list; what is not a number counts as -infinity.
template <typename T> __device__ __noinline__ Best best_slowly(const T* x, int lo, int hi, int k, int warp, int warps, int lane) {
    Best best = {-INFINITY, NO_ID};
    for (int b = lo + warp * 32; b < hi; b += 32 * warps) {
        const int i = b + lane;
        Best c = {-INFINITY, NO_ID};
        if (i < hi) {
            const float v = to_f32(x[i]);
            c = {v == v ? v : -INFINITY, i};
        }
        uint32_t lanes = __ballot_sync(0xffffffffu, better(c, shfl(best, k - 1)));
        while (lanes) {
            const Best n = shfl(c, __ffs(lanes) - 1);
            lanes &= lanes - 1;
            const uint32_t behind = __ballot_sync(0xffffffffu, better(n, best));
            if (!behind) continue;
            const int pos = __ffs(behind) - 1;
            const Best up = {__shfl_up_sync(0xffffffffu, best.v, 1), __shfl_up_sync(0xffffffffu, best.i, 1)};
            if (lane == pos) best = n;
            if (lane > pos) best = up;
        }
    }
    return best;
}

// ln of a sum of terms, the largest of which is 2^-8 at least: the exponent's part exact, the rest below ln 2
__device__ __forceinline__ double log_of(float sum) {
    if (!(sum < INFINITY)) return NAN;
    const int e = ((__float_as_int(sum) >> 23) & 255) - 127;
    return e * 0.69314718055994530942 + (double)logf(__int_as_float(__float_as_int(sum) - (e << 23)));
}
// Differences of a logit and what its row's sum says are of 64 bits: either may be large and both rounded, where only their difference counts.
__device__ __forceinline__ float log_prob(float x, double2 lse) { return (float)(((double)x - lse.x) - lse.y); }

// What is known of a row: results, and the log probabilities of tokens that are asked of it.  A whole CTA; st, best: warp 0's.
template <typename T, bool TOP, int THREADS> __device__ __forceinline__ void finish_row(const LogProbsParams& p, double2& shared_lse, const T* x, int row, Stat st, Best best) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp == 0) {
        // The sum is that of 2^(LOG2E x - m), LOG2E being the fp32 number: m / LOG2E is the reference in the logits' units, and the rounding of neither product nor
        // constant is left in it (m ln 2 in fp32 was 4e-5 off next to 1000, 5e-3 next to 10^5)
        double2 lse = {(double)st.m * (1.0 / (double)LOG2E), log_of(st.l)};
        float entropy = (float)(lse.y - (double)(st.a / st.l) * (1.0 / (double)LOG2E));
        // Nothing above the floor, or nothing that can be scaled: a row of lowest values (uniform over them), of nothing but excluded tokens, of
        // the largest values, of infinity.  Walked again as the formulas say.
        if (st.m <= floor_of<T>() * LOG2E || st.m >= L_HIGHEST) {
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
            lse = {(double)high, (double)logf(sum)};
            entropy = (float)(lse.y - (double)(weighted / sum));
            if (__any_sync(0xffffffffu, nan) || high == -INFINITY) lse.x = lse.y = entropy = NAN;
        }
        if (lane == 0) {
            p.entropy[row] = entropy;
            shared_lse = lse;
            if (!p.tokens_here) p.lse[row] = lse;
        }
        if (TOP && lane < p.top) {
            p.top_ids[(int64_t)row * p.top + lane] = best.i;
            p.top_log_probs[(int64_t)row * p.top + lane] = log_prob(best.v, lse);
        }
    }
    if (p.tokens_here && p.n_tokens > 0) {
        __syncthreads();
        const double2 lse = shared_lse;
        auto one = [&](int i) {
            const int token = p.tokens[i];
            p.log_probs[i] = token == -1 ? 0.f : (token >= 0 && token < p.vocab ? log_prob(to_f32(x[token]), lse) : NAN);
        };
        if (!p.rows) {
            if (threadIdx.x == 0) one(row);
        } else {
            for (int i = threadIdx.x; i < p.n_tokens; i += THREADS) {
                const int r = p.rows[i];
                if (r == row) one(i);
                if (row == 0 && (r < 0 || r >= p.n_rows)) p.log_probs[i] = NAN;
            }
        }
    }
}

// A stretch of a row: vectors v0 .. v1 of the whole ones behind `head` logits, and the logits around them at the row's ends
template <typename T> struct Stretch {
    const T* x;
    int row, head, n_vec, v0, v1;
    bool first, last;  // the row begins here, ends here
    __device__ __forceinline__ Stretch(const LogProbsParams& p, int r) : row(r) {
        x = static_cast<const T*>(p.logits) + (int64_t)r * p.row_stride;
        head = min(p.vocab, (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)));
        n_vec = (p.vocab - head) / Vec<T>::N;
    }
    __device__ __forceinline__ const T* at(int vec) const { return x + head + (int64_t)vec * Vec<T>::N; }
};

// CLUSTER: a cluster of CTAs has a row, CTA 0 finishes it.  Else the GPU's CTAs have equal stretches of all rows laid end to end, in turns of
// L_STEP vectors; what a stretch of a row gives goes to `parts` (number: row + CTA), and finish_rows_kernel does the rest.
//
// Logits come through a ring of three stages of 16 KiB a CTA, by 1-D bulk copies that thread 0 asks for two turns ahead: 128 KiB on their way to an
// SM, which asks nothing of registers or of the other threads, and the next row's first turns arrive while one is finished.  (Loaded to registers, a
// turn ahead, 64 KiB: 303 MB of bf16 rows of 128000 63 us.)
template <typename T, bool TOP, bool CLUSTER>
__global__ void __launch_bounds__(L_THREADS, 4) log_probs_kernel(const LogProbsParams p) {
    constexpr int N = Vec<T>::N;
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ Shared sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int S = p.splits, k = max(1, p.top);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    int64_t turn_at = 0, turn_end = 1;
    if (!CLUSTER) {
        turn_at = p.begin(blockIdx.x);
        turn_end = p.begin(blockIdx.x + 1);
    }
    auto stretch = [&](int64_t at) {
        if (CLUSTER) {
            Stretch<T> s(p, blockIdx.x / S);
            const int part = blockIdx.x % S;
            s.v0 = (int)((int64_t)s.n_vec * part / S);
            s.v1 = (int)((int64_t)s.n_vec * (part + 1) / S);
            s.first = part == 0;
            s.last = part == S - 1;
            return s;
        }
        const int row = (int)(at / p.turns), t0 = (int)(at - (int64_t)row * p.turns), t1 = (int)min((int64_t)p.turns, turn_end - (int64_t)row * p.turns);
        Stretch<T> s(p, row);
        s.v0 = min(s.n_vec, t0 * L_STEP);
        s.v1 = t1 == p.turns ? s.n_vec : min(s.n_vec, t1 * L_STEP);
        s.first = t0 == 0;
        s.last = t1 == p.turns;
        return s;
    };
    const uint32_t full = ptx::smem_u32(sh.full), empty = ptx::smem_u32(sh.empty), stages = ptx::smem_u32(ring);
    if (turn_at >= turn_end) return;
    if (tid == 0) {
        for (int i = 0; i < L_STAGES; i++) {
            ptx::mbar_init(full + 8 * i, 1);
            ptx::mbar_init(empty + 8 * i, L_WARPS);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    // Every wait is bounded: on expiry the status is recorded, no later one waits, and thread 0 sees its copies in flight land
    long long patience = L_WAIT_LIMIT;
    auto wait = [&](uint32_t bar, int parity) {
        if (ptx::mbar_wait_bounded(bar, parity, patience)) return;
        patience = 0;
        atomicCAS(&g_log_probs_status, STATUS_OK, STATUS_FULL_WAIT_TIMEOUT);
    };
    Stretch<T> s = stretch(turn_at);
    // thread 0: turns that are asked for, over all stretches
    Stretch<T> ahead = s;
    int ahead_b = s.v0, asked = 0;
    bool ahead_more = true;
    auto ask = [&] {
        while (ahead_more && ahead_b >= ahead.v1) {
            const int64_t at = ((int64_t)ahead.row + 1) * p.turns;
            ahead_more = !CLUSTER && at < turn_end;
            if (ahead_more) {
                ahead = stretch(at);
                ahead_b = ahead.v0;
            }
        }
        if (!ahead_more) return;
        const int stage = asked % L_STAGES, bytes = min(L_STEP, ahead.v1 - ahead_b) * 16;
        if (asked >= L_STAGES) wait(empty + 8 * stage, (asked / L_STAGES - 1) & 1);
        ptx::mbar_arrive_expect_tx(full + 8 * stage, bytes);
        ptx::bulk_copy_g2s(stages + stage * L_STEP * 16, ahead.at(ahead_b), bytes, full + 8 * stage);
        ahead_b += L_STEP;
        asked++;
    };
    auto drain = [&] {
        if (tid == 0 && patience == 0)
            for (int i = max(0, asked - L_STAGES); i < asked; i++) ptx::mbar_wait_bounded(full + 8 * (i % L_STAGES), (i / L_STAGES) & 1, L_WAIT_LIMIT);
    };
    if (tid == 0) {
        ask();
        ask();
    }
    if (TOP) {
        for (int i = tid; i < L_ROWS * L_GROUPS; i += L_THREADS) sh.group[i / L_GROUPS][i % L_GROUPS] = -INFINITY;
        if (tid < L_ROWS) sh.n_hits[tid] = 0;
        if (tid == 0) sh.n_found = 0;
        __syncthreads();
    }
    int taken = 0;  // turns
    for (int n = 0;; n++) {
        // What is shared of row n is in place n % 3.  Place (n + 1) % 3 was row n - 2's, which every warp has left when this one has met the
        // others at the end of row n - 1; nobody is at row n + 1 before they meet at the end of this one.
        const int place = n % L_ROWS;
        if (TOP && n > 1) {
            const int clear = (n + 1) % L_ROWS;
            if (tid < L_GROUPS) sh.group[clear][tid] = -INFINITY;
            if (tid == 0) sh.n_hits[clear] = 0;
        }
        Sums sums;
        float mine = -INFINITY;  // this thread's largest
        auto tell = [&] {  // the group's largest
            float high = fmaxf(mine, __shfl_xor_sync(0xffffffffu, mine, 1));
            if (wide_groups(k)) {
                high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, 2));
                if ((lane & 3) == 0) *const_cast<volatile float*>(&sh.group[place][warp * 8 + (lane >> 2)]) = high;
            } else if ((lane & 1) == 0) {
                *const_cast<volatile float*>(&sh.group[place][warp * 16 + (lane >> 1)]) = high;
            }
        };
        float limit = least_of<T>();
        int turn = 0;
        auto work = [&](int b, auto whole) {
            constexpr bool WHOLE = decltype(whole)::value;  // no vector is behind the stretch's end
            const int stage = taken % L_STAGES;
            if (tid == 0) ask();  // into the stage of the turn before
            wait(full + 8 * stage, (taken / L_STAGES) & 1);
            Vec<T> v[L_UNROLL];
#pragma unroll
            for (int u = 0; u < L_UNROLL; u++) v[u].load_shared(stages + (stage * L_STEP + u * L_THREADS + tid) * 16);
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(empty + 8 * stage);
            taken++;
            uint32_t high[L_UNROLL], both = Vec<T>::NOTHING;
#pragma unroll
            for (int u = 0; u < L_UNROLL; u++) {
                high[u] = Vec<T>::NOTHING;
                if (WHOLE || b + u * L_THREADS + tid < s.v1) high[u] = v[u].lift();
                both = Vec<T>::larger(both, high[u]);
            }
            const float highest = Vec<T>::value(both);
            if (TOP) {
                mine = fmaxf(mine, highest);
                // from the first turn, for which the warps wait for one another, and again after 4, 16 ..., from what has been told
                if (((turn + 1) & turn) == 0 && ((turn + 1) & 0x55555555)) {
                    tell();
                    if (turn == 0) __syncthreads();
                    else __syncwarp();
                    limit = fmaxf(limit, kth_of_groups(sh.group[place], k, lane));
                }
                if (highest >= limit) {
                    // Only noted: looked at here, the code for it, little used and seldom where it was read, took 2.7 us each time
                    uint32_t vectors = 0;
#pragma unroll
                    for (int u = 0; u < L_UNROLL; u++) vectors |= (Vec<T>::value(high[u]) >= limit ? 1u : 0u) << u;
                    const int at = atomicAdd(&sh.n_hits[place], 1);
                    if (at < L_HITS) sh.hits[place][at] = note_of(turn, tid, vectors);
                }
                __syncwarp();  // together again: else the sums below are gone through lane by lane
            }
            sums.move(fmaxf(highest, floor_of<T>()));
#pragma unroll
            for (int u = 0; u < L_UNROLL; u++) {
                if (!WHOLE && b + u * L_THREADS + tid >= s.v1) continue;
                float f[N];
                v[u].get(f);
                sums.add(f);
            }
            turn++;
        };
        for (int b = s.v0; b < s.v1; b += L_STEP) {
            if (b + L_STEP <= s.v1) work(b, std::true_type());
            else work(b, std::false_type());
        }
        // the logits outside of whole vectors, one a lane
        const int tail = p.vocab - s.head - s.n_vec * N;
        const int odd = s.first && warp == 0 && lane < s.head ? lane : (s.last && warp == L_WARPS - 1 && lane < tail ? p.vocab - tail + lane : -1);
        if (odd >= 0) sums.add_one(to_f32(s.x[odd]), floor_of<T>());

        // ---- lanes, warps
        Stat st = sums.total();
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1)
            st = join(st, {__shfl_xor_sync(0xffffffffu, st.m, off), __shfl_xor_sync(0xffffffffu, st.l, off), __shfl_xor_sync(0xffffffffu, st.a, off)});
        if (lane == 0) sh.stat[place][warp] = st;
        if (TOP) tell();
        __syncthreads();
        auto joined = [&] {  // of the warps
            Stat w = sh.stat[place][lane & (L_WARPS - 1)];
#pragma unroll
            for (int off = L_WARPS / 2; off >= 1; off >>= 1)
                w = join(w, {__shfl_xor_sync(0xffffffffu, w.m, off), __shfl_xor_sync(0xffffffffu, w.l, off), __shfl_xor_sync(0xffffffffu, w.a, off)});
            return w;
        };
        if (!CLUSTER) {
            // The rest is another kernel's, for all rows together: here the CTA's chain of syncs and reads (about 4 us a row) would stand
            // between it and the next row
            LogProbsPart& to = p.parts[(int64_t)s.row + blockIdx.x];
            if (warp == 0) {
                st = joined();
                if (lane == 0) {
                    to.m = st.m;
                    to.l = st.l;
                    to.a = st.a;
                }
            }
            if (TOP) {
                const int hits = sh.n_hits[place];
                if (warp == 1) {
                    const float last = fmaxf(least_of<T>(), kth_of_groups(sh.group[place], k, lane));
                    if (lane == 0) {
                        to.limit = last;
                        to.n_hits = hits;
                    }
                }
                uint32_t* const notes = p.hits + ((int64_t)s.row + blockIdx.x) * p.hits_room;
                for (int i = tid; i < min(hits, p.hits_room); i += L_THREADS) notes[i] = sh.hits[place][i];
            }
            turn_at = ((int64_t)s.row + 1) * p.turns;
            if (turn_at >= turn_end) {
                drain();
                return;
            }
            s = stretch(turn_at);
            continue;
        }

        // ---- a cluster finishes its row
        drain();
        Best best = {-INFINITY, NO_ID};
        if (TOP) {
            const int lo = s.first ? 0 : s.head + s.v0 * N, hi = s.last ? p.vocab : s.head + s.v1 * N, hits = sh.n_hits[0];
            limit = fmaxf(least_of<T>(), kth_of_groups(sh.group[0], k, lane));
            auto keep = [&](float v, int id) {
                const int at = atomicAdd(&sh.n_found, 1);
                if (at < L_FOUND) sh.one.found[at] = {v, id};
            };
            if (hits <= L_HITS) look_at(s.x + s.head, s.head, s.v0, sh.one.own, hits, limit, tid, L_THREADS, keep);
            if (odd >= 0 && to_f32(s.x[odd]) >= limit) keep(to_f32(s.x[odd]), odd);
            if (warp == 0) sh.one.list[0][lane] = {-INFINITY, NO_ID};
            __syncthreads();
            const int found = sh.n_found;
            if (hits > L_HITS || found > L_FOUND || found < min(k, hi - lo)) {
                best = best_slowly(s.x, lo, hi, k, warp, L_WARPS, lane);
                sh.one.list[warp][lane] = best;
#pragma unroll
                for (int half = L_WARPS / 2; half >= 1; half >>= 1) {
                    __syncthreads();
                    if (warp < half) sh.one.list[warp][lane] = best = merge_lists(best, sh.one.list[warp + half][lane], lane);
                }
            } else {
                put_in_order(sh.one.found, found, sh.one.list[0], tid, L_THREADS);
                __syncthreads();
                if (warp == 0) best = sh.one.list[0][lane];
            }
        }
        if (warp == 0) st = joined();
        if (S > 1) {
            __syncwarp();
            if (warp == 0 && lane == 0) sh.stat[0][0] = st;
            if (TOP && warp == 0) sh.one.list[0][lane] = best;
            asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
            asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
            if (s.first && warp == 0) {
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
                const uint32_t a = remote(&sh.stat[0][0], lane & (S - 1));
                st = {__uint_as_float(read(a)), __uint_as_float(read(a + 4)), __uint_as_float(read(a + 8))};
                for (int off = S / 2; off >= 1; off >>= 1)
                    st = join(st, {__shfl_xor_sync(0xffffffffu, st.m, off), __shfl_xor_sync(0xffffffffu, st.l, off), __shfl_xor_sync(0xffffffffu, st.a, off)});
                if (TOP) {
                    Best other[8];
#pragma unroll
                    for (int r = 0; r < 8; r++) {
                        other[r] = {-INFINITY, NO_ID};
                        if (r < S) {
                            const uint32_t b = remote(&sh.one.list[0][lane], r);
                            other[r] = {__uint_as_float(read(b)), (int)read(b + 4)};
                        }
                    }
#pragma unroll
                    for (int half = 4; half >= 1; half >>= 1)
#pragma unroll
                        for (int r = 0; r < half; r++) other[r] = merge_lists(other[r], other[r + half], lane);
                    best = other[0];
                }
            }
            asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
            asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
            if (!s.first) return;
        }
        finish_row<T, TOP, L_THREADS>(p, sh.lse, s.x, s.row, st, best);
        return;
    }
}

// The rows of which log_probs_kernel has left parts: a CTA for every row
template <typename T, bool TOP>
__global__ void __launch_bounds__(F_THREADS) finish_rows_kernel(const LogProbsParams p, int n_ctas) {
    __shared__ Best found[L_FOUND], list[F_WARPS][32];
    __shared__ int n_found;
    __shared__ double2 lse;
    const int row = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, k = max(1, p.top);
    // the stretches of CTAs b0 .. b1: the one in which the row begins and those that begin inside it
    const int64_t row_begin = (int64_t)row * p.turns;
    const int b0 = p.owner(row_begin), b1 = min(n_ctas - 1, p.owner(row_begin + p.turns - 1));
    if (TOP) {
        if (tid == 0) n_found = 0;
        list[warp][lane] = {-INFINITY, NO_ID};
        __syncthreads();
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const Stretch<T> s(p, row);
    Stat st = {-3.0e38f, 0.f, 0.f};
    float limit = least_of<T>();
    bool many = false;
    for (int b = b0; b <= b1; b++) {
        const LogProbsPart& from = p.parts[(int64_t)row + b];
        const Stat one = {from.m, from.l, from.a};
        if (TOP) {
            limit = fmaxf(limit, from.limit);
            many = many || from.n_hits > p.hits_room;
        }
        st = join(st, one);
    }
    Best best = {-INFINITY, NO_ID};
    if (TOP) {
        auto keep = [&](float v, int id) {
            const int at = atomicAdd(&n_found, 1);
            if (at < L_FOUND) found[at] = {v, id};
        };
        if (!many)
            for (int b = b0; b <= b1; b++) {
                const LogProbsPart& from = p.parts[(int64_t)row + b];
                look_at(s.x + s.head, s.head, min(s.n_vec, (int)max((int64_t)0, p.begin(b) - row_begin) * L_STEP), p.hits + ((int64_t)row + b) * p.hits_room, from.n_hits, limit, tid, F_THREADS, keep);
            }
        const int around = s.head + (p.vocab - s.head - s.n_vec * Vec<T>::N);  // logits outside of whole vectors
        if (tid < around) {
            const int id = tid < s.head ? tid : p.vocab - around + tid;
            const float f = to_f32(s.x[id]);
            if (f >= limit) keep(f, id);
        }
        __syncthreads();
        const int n = n_found;
        if (many || n > L_FOUND || n < min(k, p.vocab)) {
            best = best_slowly(s.x, 0, p.vocab, k, warp, F_WARPS, lane);
            list[warp][lane] = best;
#pragma unroll
            for (int half = F_WARPS / 2; half >= 1; half >>= 1) {
                __syncthreads();
                if (warp < half) list[warp][lane] = best = merge_lists(best, list[warp + half][lane], lane);
            }
        } else {
            put_in_order(found, n, list[0], tid, F_THREADS);
            __syncthreads();
            best = list[0][lane];
        }
    }
    finish_row<T, TOP, F_THREADS>(p, lse, s.x, row, st, best);
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
        const double2 lse = p.lse[row];
        if (token >= 0 && token < p.vocab) lp = log_prob(to_f32(static_cast<const T*>(p.logits)[(int64_t)row * p.row_stride + token]), lse);
        if (token == -1) lp = 0.f;
    }
    p.log_probs[i] = lp;
}

template <typename T>
cudaError_t launch(const LogProbsParams& p, cudaStream_t stream) {
    auto with_ring = [](auto* k) { return allow_shared(reinterpret_cast<const void*>(k), L_RING); };
    if (p.n_rows > 0) {
        cudaError_t e;
        if (p.splits > 0) {
            auto* k = p.top > 0 ? &log_probs_kernel<T, true, true> : &log_probs_kernel<T, false, true>;
            e = with_ring(k);
            if (e == cudaSuccess) e = launch_kernel(k, dim3((unsigned)(p.n_rows * p.splits)), L_THREADS, L_RING, p.splits, true, stream, p);
        } else {
            const int ctas = log_probs_ctas();
            auto* k = p.top > 0 ? &log_probs_kernel<T, true, false> : &log_probs_kernel<T, false, false>;
            auto* j = p.top > 0 ? &finish_rows_kernel<T, true> : &finish_rows_kernel<T, false>;
            e = with_ring(k);
            if (e == cudaSuccess) e = launch_kernel(k, dim3((unsigned)ctas), L_THREADS, L_RING, 1, true, stream, p);
            if (e == cudaSuccess) e = launch_kernel(j, dim3((unsigned)p.n_rows), F_THREADS, 0, 1, true, stream, p, ctas);
        }
        if (e != cudaSuccess) return e;
    }
    if (p.n_tokens > 0 && !p.tokens_here) return launch_kernel(&given_tokens_kernel<T>, dim3((unsigned)((p.n_tokens + 127) / 128)), 128, 0, 1, true, stream, p);
    return cudaSuccess;
}

int turns_of(int vocab, int esize) { return std::max(1, (vocab / (16 / esize) + L_STEP - 1) / L_STEP); }

}  // namespace

int log_probs_ctas() { return 4 * B200_SMS; }

// CTAs of a row's cluster, or 0: rows enough to hand out stretches of, a few turns at least to every CTA
int log_probs_splits(int n_rows, int vocab, int esize) {
    if ((int64_t)n_rows * turns_of(vocab, esize) >= 3 * log_probs_ctas() && n_rows > log_probs_ctas() / 8) return 0;
    int s = 1;
    while (s < 8 && (int64_t)n_rows * s * 2 <= log_probs_ctas() && (int64_t)vocab * esize / s >= 16384) s *= 2;
    return s;
}

// A note is of one whole vector at least: short rows cannot have more of them
int log_probs_hits_room(int vocab, int esize) { return std::min(L_HITS, std::max(1, vocab / (16 / esize))); }

void log_probs_shape(LogProbsParams& p, int esize) {
    p.hits_room = log_probs_hits_room(p.vocab, esize);
    p.splits = log_probs_splits(p.n_rows, p.vocab, esize);
    p.turns = turns_of(p.vocab, esize);
    const int64_t all = (int64_t)p.n_rows * p.turns;
    p.each = all / log_probs_ctas();
    p.more = (int)(all % log_probs_ctas());
}

cudaError_t read_log_probs_status(int* status, cudaStream_t stream) {
    cudaError_t e = cudaMemcpyFromSymbolAsync(status, g_log_probs_status, sizeof(int), 0, cudaMemcpyDeviceToHost, stream);
    return e == cudaSuccess ? cudaStreamSynchronize(stream) : e;
}

cudaError_t launch_log_probs(const LogProbsParams& p, int dtype, cudaStream_t stream) {
    if (dtype == CA_DTYPE_F32) return launch<float>(p, stream);
    if (dtype == CA_DTYPE_F16) return launch<__half>(p, stream);
    return launch<__nv_bfloat16>(p, stream);
}

}  // namespace ca
