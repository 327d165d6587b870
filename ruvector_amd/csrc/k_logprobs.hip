// k_logprobs.hip — log probabilities of given ids over rows of scores, with rank, entropy and
// the best alternatives, in one pass over the scores; and the gradient by the scores.
//
// With u = (s - m) / T, m the row's largest score, S = sum e^u and E = sum e^u u:
//   log p_t = u_t - ln S,   H = -sum p ln p = ln S - E / S.
// m, S and E over a part of a row join with those over another part (m' = max, S' = S r + ..,
// E' = r (E + S d) + .. with d = (m - m') / T, r = e^d), so one pass suffices. All three are
// kept in 32 bits, in units of log2, for v_exp_f32.
//
// It cannot do without one read of the scores. bf16 8192 x 32000: 97 us (5.4 TB/s) for log p and the statistics,
// 111 to 137 with rank, entropy and the best 5; f32 2503 x 10007: 17 and 31 us (the best 10). The difference
// is instructions: rank, entropy and candidates take as many again as the sum. 35 us with a tenth of the scores
// masked: with the entropy, a step that holds a masked score takes its products twice.
#include "heads.hpp"

namespace rvx {
namespace {

constexpr float LN2 = 0.69314718055994530942f, LOG2E = 1.44269504088896340736f;
constexpr float FLOOR_U = -1e4f;   // 2^u is 0 long before; keeps 0 * u finite for masked scores
constexpr float FAR_U = 67108864.0f;  // 2^26: past it fl(m c1) may be off by more than 2^u can take
using u64 = unsigned long long;

struct Stat {
    float m = -3.402823466e38f, s = 0.f, e = 0.f;
};
__device__ __forceinline__ Stat join(const Stat& a, const Stat& b, float c1) {
    Stat o;
    o.m = fmaxf(a.m, b.m);
    const float da = fmaxf((a.m - o.m) * c1, FLOOR_U), db = fmaxf((b.m - o.m) * c1, FLOOR_U);
    const float ra = __builtin_amdgcn_exp2f(da), rb = __builtin_amdgcn_exp2f(db);
    o.s = fmaf(a.s, ra, b.s * rb);
    o.e = fmaf(ra, fmaf(a.s, da, a.e), rb * fmaf(b.s, db, b.e));
    return o;
}

// ---------------------------------------------------------------- values of other lanes
// The lane number, hidden from the compiler: masks made from it stay where they are used. (Hoisted
// out of the loops around, a sort's masks overflow the scalar registers.)
__device__ __forceinline__ int local_lane() {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    return lane;
}
// x of lane (l ^ ST), without a trip through LDS: rows of 16 lanes are permuted by DPP, rows and
// halves exchanged by the permlane swaps.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
}
template <int ST>
__device__ __forceinline__ uint32_t lane_xor(uint32_t x) {
    if constexpr (ST == 1) return dpp<0xB1>(x);             // quad_perm [1,0,3,2]
    else if constexpr (ST == 2) return dpp<0x4E>(x);        // quad_perm [2,3,0,1]
    else if constexpr (ST == 4) return dpp<0x1B>(dpp<0x141>(x));  // mirror of 8 lanes, then of 4: l ^ 7 ^ 3
    else if constexpr (ST == 8) return dpp<0x128>(x);       // rotation of a row by 8
    else if constexpr (ST == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
        return local_lane() & 16 ? r[0] : r[1];
    } else {
        const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        return local_lane() & 32 ? r[0] : r[1];
    }
}
template <int ST>
__device__ __forceinline__ float lane_xor(float x) {
    return __uint_as_float(lane_xor<ST>(__float_as_uint(x)));
}
template <int ST>
__device__ __forceinline__ u64 lane_xor(u64 x) {
    return (u64)lane_xor<ST>((uint32_t)(x >> 32)) << 32 | lane_xor<ST>((uint32_t)x);
}
// One exchange of a bitonic network: the smaller value goes to the lower lane where `up`.
template <int ST, class K>
__device__ __forceinline__ K exchange(K x, bool up, int lane) {
    const K y = lane_xor<ST>(x);
    return ((lane & ST) == 0) == up == (x < y) ? x : y;
}
template <int SIZE, int ST, class K>
__device__ __forceinline__ K sort_stage(K x, int lane) {  // the stage of SIZE: strides ST, ST / 2 .. 1
    x = exchange<ST>(x, (lane & SIZE) == 0, lane);
    if constexpr (ST > 1) x = sort_stage<SIZE, ST / 2>(x, lane);
    return x;
}
template <class K>
__device__ __forceinline__ K sort_up(K x) {  // ascending over the 64 lanes
    const int lane = local_lane();
    x = sort_stage<2, 1>(x, lane);
    x = sort_stage<4, 2>(x, lane);
    x = sort_stage<8, 4>(x, lane);
    x = sort_stage<16, 8>(x, lane);
    x = sort_stage<32, 16>(x, lane);
    return sort_stage<64, 32>(x, lane);
}
template <int ST = 32>
__device__ __forceinline__ u64 bitonic_down(u64 x, int lane) {  // a bitonic row to descending order
    x = exchange<ST>(x, false, lane);
    if constexpr (ST > 1) x = bitonic_down<ST / 2>(x, lane);
    return x;
}
__device__ __forceinline__ Stat join_lanes(Stat st, float c1) {
    auto step = [&](auto o) {
        constexpr int ST = decltype(o)::value;
        Stat b;
        b.m = lane_xor<ST>(st.m), b.s = lane_xor<ST>(st.s), b.e = lane_xor<ST>(st.e);
        st = join(st, b, c1);
    };
    step(std::integral_constant<int, 32>{});
    step(std::integral_constant<int, 16>{});
    step(std::integral_constant<int, 8>{});
    step(std::integral_constant<int, 4>{});
    step(std::integral_constant<int, 2>{});
    step(std::integral_constant<int, 1>{});
    return st;
}

// ---------------------------------------------------------------- the best scores
// Scores in the order "higher first, then lower id first", as 64-bit keys (0 = none).
__device__ __forceinline__ u64 key_of(float x, uint32_t id) {
    int b = __float_as_int(x + 0.0f);  // -0 and +0 are the same score
    b ^= (b >> 31) & 0x7fffffff;
    return ((u64)((uint32_t)b ^ 0x80000000u) << 32) | (0xffffffffu - id);
}
__device__ __forceinline__ float key_score(u64 k) {
    int b = (int)((uint32_t)(k >> 32) ^ 0x80000000u);
    b ^= (b >> 31) & 0x7fffffff;
    return __int_as_float(b);
}
__device__ __forceinline__ u64 lane_value(u64 x, int lane) {  // lane: the same in all lanes
    return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)x, lane);
}

// The k best keys a wave has seen, one a lane, best first. Keys above the k-th best wait in LDS until
// some of them are merged:
// k <= 8: the list's and the waiting keys each look how many of all are larger: their place. That is
// 3 instructions a key, a few keys at a time.
// k > 8: 64 waiting keys are sorted (bitonic, ascending) and merged: max(best, new) of a descending
// and an ascending row holds the 64 largest as a bitonic row.
struct Best {
    static constexpr int ROOM = 192;  // 63 waiting and 64 offered at once (k <= 8: less, and 8 of the list); 64 places
    u64 list = 0, tau = 0;  // tau: no key up to it can be among the k best
    float tau_score = -INFINITY;
    int waiting = 0, k;
    u64* pend;
    __device__ Best(u64* p, int kk) : k(kk), pend(p) {}

    __device__ __forceinline__ void tighten() {
        const u64 kth = lane_value(list, k - 1);
        if (kth > tau) {
            tau = kth;
            tau_score = key_score(tau);
        }
    }
    // At least k scores are known to be `bound` or above (-inf: nothing is known).
    __device__ __forceinline__ void bound(float score) {
        if (score > -INFINITY) {
            tau = key_of(score, 0xffffffffu);
            tau_score = score;
        }
    }
    __device__ __forceinline__ void flush() {  // the last waiting keys, as many as go at once
        const int lane = threadIdx.x & 63;
        if (k <= 8) {
            const int from = max(0, waiting - (64 - k)), total = waiting - from + k;
            if (lane < k) pend[waiting + lane] = list;
            wave_lds_order();
            const u64* all = pend + from;
            const u64 own = lane < total ? all[lane] : 0;
            int place = 0;
#pragma unroll 4
            for (int j = 0; j < total; ++j) place += all[j] > own ? 1 : 0;
            const int there = __popcll(__ballot(own != 0));
            if (own != 0 && place < k) pend[128 + place] = own;
            wave_lds_order();
            list = lane < min(k, there) ? pend[128 + lane] : 0;
            waiting = from;
            tighten();
        } else {
            wave_lds_order();
            const int from = max(0, waiting - 64);
            u64 x = from + lane < waiting ? pend[from + lane] : 0;
            waiting = from;
            if (!__any(x > tau)) return;
            take(sort_up(x));
        }
    }
    __device__ __forceinline__ void take(u64 ascending) {
        list = bitonic_down(list > ascending ? list : ascending, local_lane());
        tighten();
    }
    __device__ __forceinline__ void offer(u64 key, bool there) {
        const bool in = there && key > tau;
        const u64 mask = __ballot(in);
        if (in)
            pend[waiting + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                                     __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0))] = key;
        waiting += __popcll(mask);
    }
    // Waiting keys are merged once they are worth it: a late tau lets more scores through.
    __device__ __forceinline__ void settle() {
        const int worth = k <= 8 ? 16 : 64;
        while (waiting >= worth) flush();
    }
};

struct Part {  // what one block found of one row
    float m, s, e;
    int before;
};

// (score - m) / T; halves, as the difference itself may be past the largest float
__device__ __forceinline__ float gap(float score, float m, float temp) {
    return 2.0f * ((0.5f * score - 0.5f * m) / temp);
}
__device__ __forceinline__ void write_row(const Stat& st, int before, int64_t row, float st_score, bool has_target,
                                          float temp, const LogProbsOut& out) {
    const bool empty = st.s == 0.0f;
    const float m = empty ? -INFINITY : st.m;
    const float log_sum = empty ? -INFINITY : logf(st.s);
    if (out.logp) out.logp[row] = !has_target ? 0.0f : empty ? -INFINITY : gap(st_score, m, temp) - log_sum;
    if (out.rank) out.rank[row] = has_target ? before : -1;
    if (out.entropy) out.entropy[row] = empty ? 0.0f : log_sum - LN2 * (st.e / st.s);
    if (out.stats) {
        out.stats[2 * row] = m;
        out.stats[2 * row + 1] = log_sum;
    }
}
__device__ __forceinline__ void write_top(u64 list, int k, int64_t row, const Stat& st, float temp,
                                          const LogProbsOut& out) {
    const int lane = threadIdx.x & 63;
    if (lane >= k) return;
    const bool none = list == 0;
    if (out.top_ids) out.top_ids[row * k + lane] = none ? -1 : (int64_t)(0xffffffffu - (uint32_t)list);
    if (out.top_logp)
        out.top_logp[row * k + lane] = none ? -INFINITY : gap(key_score(list), st.m, temp) - logf(st.s);
}

// ---------------------------------------------------------------- one pass
constexpr int LP_U = 2, LP_WAVES = 4;  // 16-byte loads per lane and step; waves per block

// A wave's elements of one step, 16 bytes a lane and load. In a row's last step a lane whose piece
// would pass the end takes the row's last piece, and drops what is not its own: no lane branches.
template <class T>
struct Step {
    static constexpr int N = Vec16<T>::N, SIZE = 64 * N * LP_U;
    Vec16<T> v[LP_U];
    static __device__ __forceinline__ int place(int u, int64_t left) {  // the piece's begin, from the step's on
        const int p = (u * 64 + (threadIdx.x & 63)) * N;
        return left >= SIZE ? p : (int)min((int64_t)p, left - N);
    }
    __device__ __forceinline__ void load(const T* x, int64_t at, int64_t hi) {
        if (hi < N) {  // a row shorter than a piece: every lane holds it
#pragma unroll
            for (int u = 0; u < LP_U; ++u)
#pragma unroll
                for (int j = 0; j < N; ++j) v[u].v[j] = j >= N - hi ? x[j - (N - hi)] : (T)-INFINITY;
            return;
        }
#pragma unroll
        for (int u = 0; u < LP_U; ++u) v[u] = load16(x + at + place(u, hi - at));
    }
    __device__ __forceinline__ void values(float (&f)[LP_U][N], int64_t left) const {
#pragma unroll
        for (int u = 0; u < LP_U; ++u)
#pragma unroll
            for (int j = 0; j < N; ++j) f[u][j] = (float)v[u].v[j];
        if (left >= SIZE) return;
#pragma unroll
        for (int u = 0; u < LP_U; ++u) {
            const int drop = (u * 64 + (int)(threadIdx.x & 63)) * N - place(u, left);
#pragma unroll
            for (int j = 0; j < N; ++j) f[u][j] = j < drop ? -INFINITY : f[u][j];
        }
    }
};

// S and E by subtraction of the running maximum itself: right for scores of any size. Only where a
// row's largest |score| / T is past FAR_U.
template <class T>
__device__ __attribute__((noinline)) Stat far_stats(const T* x, int64_t lo, int64_t hi, float c1) {
    Stat st;
#pragma unroll 1
    for (int64_t i = lo + (threadIdx.x & 63); i < hi; i += 64) {
        const float v = (float)x[i], mn = fmaxf(st.m, v);
        const float d = fmaxf((st.m - mn) * c1, FLOOR_U), r = __builtin_amdgcn_exp2f(d);
        const float y = (v - mn) * c1, ex = __builtin_amdgcn_exp2f(y);
        st.e = fmaf(r, fmaf(st.s, d, st.e), ex * fmaxf(y, FLOOR_U));
        st.s = fmaf(st.s, r, ex);
        st.m = mn;
    }
    return st;
}

// A wave goes over elements [lo, hi) of a row. Bound by reading them: per score one unpack, half a
// max, one fma, one exp (4 cycles), two additions and one comparison. The next step's loads are on
// their way meanwhile; no lane branches around loads, which would serialise them.
template <class T, bool ENT, bool RANK, bool TOP>
__device__ __forceinline__ Stat walk(const T* __restrict__ x, int64_t lo, int64_t hi, float c1, int64_t target,
                                     float st_score, int& before, Best& best) {
    constexpr int N = Step<T>::N, SIZE = Step<T>::SIZE;
    const int lane = threadIdx.x & 63;
    // 2^u is taken against b = fl(m c1), the lane's largest score in log2 units: u = fma(x, c1, -b) is
    // rounded once, and what b is off from m c1 is put right at the end.
    const float far = fminf(FAR_U / c1, 1e30f);
    float m = -INFINITY, b = -far * c1, s = 0.f, e = 0.f;
    Step<T> nxt;
    if (lo < hi) nxt.load(x, lo, hi);
    for (int64_t at = lo; at < hi; at += SIZE) {
        float v[LP_U][N];
        nxt.values(v, hi - at);
        if (at + SIZE < hi) nxt.load(x, at + SIZE, hi);  // on its way while this step is worked on
        float cm = -INFINITY;
#pragma unroll
        for (int u = 0; u < LP_U; ++u)
#pragma unroll
            for (int j = 0; j < N; ++j) cm = fmaxf(cm, v[u][j]);
        if (__any(cm > m)) {
            m = fmaxf(m, cm);
            const float bn = fminf(fmaxf(m, -far), far) * c1;
            const float d = fmaxf(b - bn, FLOOR_U), r = __builtin_amdgcn_exp2f(d);
            if constexpr (ENT) e = r * fmaf(s, d, e);
            s *= r;
            b = bn;
        }
        float ds = 0.f, de = 0.f;
#pragma unroll
        for (int u = 0; u < LP_U; ++u)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float y = fmaf(v[u][j], c1, -b), ex = __builtin_amdgcn_exp2f(y);
                ds += ex;
                if constexpr (ENT) de = fmaf(ex, y, de);
            }
        if constexpr (ENT) {
            if (__any(de != de)) {  // a masked score (0 * -inf) or a NaN
                de = 0.f;
                float again = b;  // (hidden: or the 32 values of this path's terms are kept for it)
                asm volatile("" : "+v"(again));
#pragma unroll
                for (int u = 0; u < LP_U; ++u)
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        const float y = fmaf(v[u][j], c1, -again);
                        de = fmaf(__builtin_amdgcn_exp2f(y), fmaxf(y, FLOOR_U), de);
                    }
            }
            e += de;
        }
        s += ds;
        if constexpr (RANK) {
            if (at + SIZE <= target) {
#pragma unroll
                for (int u = 0; u < LP_U; ++u)
#pragma unroll
                    for (int j = 0; j < N; ++j) before += __popcll(__ballot(v[u][j] >= st_score));
            } else if (at > target) {
#pragma unroll
                for (int u = 0; u < LP_U; ++u)
#pragma unroll
                    for (int j = 0; j < N; ++j) before += __popcll(__ballot(v[u][j] > st_score));
            } else {
                const int t = (int)(target - at);
#pragma unroll
                for (int u = 0; u < LP_U; ++u)
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        const int place = Step<T>::place(u, hi - at) + j;  // dropped ones are not counted
                        before += __popcll(__ballot(v[u][j] > st_score || (v[u][j] == st_score && place < t &&
                                                                           place >= (u * 64 + lane) * N)));
                    }
            }
        }
        if constexpr (TOP) {
            // the k-th best of the lanes' largest scores of the first step bounds the k-th best score
            if (at == lo) best.bound(__uint_as_float(__builtin_amdgcn_readlane((int)__float_as_uint(sort_up(cm)), 64 - best.k)));
            if (at == lo || __any(cm > best.tau_score)) {
                // each lane's candidates as bits, then one of each lane at a time
                const float from = fmaxf(best.tau_score, -3.402823466e38f);
                uint32_t bits = 0;
#pragma unroll
                for (int u = 0; u < LP_U; ++u)
#pragma unroll
                    for (int j = 0; j < N; ++j) bits |= v[u][j] >= from ? 1u << (u * N + j) : 0;
                while (__any(bits != 0)) {
                    const bool has = bits != 0;
                    const int e = has ? __ffs(bits) - 1 : 0;
                    bits &= bits - 1;
                    const uint32_t pos = (uint32_t)at + Step<T>::place(e / N, hi - at) + e % N;
                    float score = v[0][0];
#pragma unroll
                    for (int i = 1; i < LP_U * N; ++i) score = e == i ? v[i / N][i % N] : score;
                    best.offer(key_of(score, pos), has);
                    best.settle();
                }
            }
        }
    }
    if constexpr (TOP)
        if (best.waiting) best.flush();
    Stat st;
    if (s != 0.f) {  // to the reference m itself; d is large only below -far, where the lane adds nothing
        const float d = fminf(fmaf(-m, c1, b), 100.0f), r = __builtin_amdgcn_exp2f(d);
        st.m = m;
        st.e = r * fmaf(s, d, e);
        st.s = s * r;
    }
    if (__any(fabsf(m) > far && m != -INFINITY)) {
        // lanes past it count only where the largest score is there too
        float mw = m;
        mw = fmaxf(mw, lane_xor<32>(mw)), mw = fmaxf(mw, lane_xor<16>(mw)), mw = fmaxf(mw, lane_xor<8>(mw));
        mw = fmaxf(mw, lane_xor<4>(mw)), mw = fmaxf(mw, lane_xor<2>(mw)), mw = fmaxf(mw, lane_xor<1>(mw));
        if (fabsf(mw) > far) st = far_stats(x, lo, hi, c1);
    }
    return join_lanes(st, c1);
}

struct Row {  // a row's target
    int64_t target;
    bool there;
    float score;
    template <class T>
    __device__ __forceinline__ Row(const T* x, const int64_t* targets, int64_t row, int64_t c) {
        target = targets ? targets[row] : -1;
        there = target >= 0 && target < c;
        if (!there) target = -1;
        score = there ? (float)x[target] : NAN;
    }
};

// A wave a row (many rows).
template <class T, bool ENT, bool RANK, bool TOP>
__global__ __launch_bounds__(64 * LP_WAVES) void logprobs_wave_kernel(const T* __restrict__ scores, int64_t n, int64_t c,
                                                                     int64_t ld, float c1, float temp,
                                                                     const int64_t* __restrict__ targets, int k,
                                                                     LogProbsOut out) {
    constexpr int ROOM = Best::ROOM;
    __shared__ u64 pend[TOP ? LP_WAVES * ROOM : 1];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = (int64_t)blockIdx.x * LP_WAVES + wave;
    if (row >= n) return;
    const T* x = scores + row * ld;
    const Row r(x, targets, row, c);
    int before = 0;
    Best best(TOP ? pend + wave * ROOM : nullptr, k);
    const Stat st = walk<T, ENT, RANK, TOP>(x, 0, c, c1, r.target, r.score, before, best);
    if ((threadIdx.x & 63) == 0) write_row(st, before, row, r.score, r.there, temp, out);
    if constexpr (TOP) write_top(best.list, k, row, st, temp, out);
}

// A block a row, or one of `splits` parts of a row: its waves take a quarter each and join in LDS.
// parts == null: the block has the whole row.
template <class T, bool ENT, bool RANK, bool TOP>
__global__ __launch_bounds__(64 * LP_WAVES) void logprobs_block_kernel(const T* __restrict__ scores, int64_t c, int64_t ld,
                                                                      float c1, float temp,
                                                                      const int64_t* __restrict__ targets, int k,
                                                                      int splits, int64_t seg_len, Part* parts, u64* keys,
                                                                      LogProbsOut out) {
    constexpr int ROOM = Best::ROOM;
    __shared__ u64 pend[TOP ? LP_WAVES * ROOM : 1];
    __shared__ Part found[LP_WAVES];
    __shared__ u64 lists[TOP ? LP_WAVES : 1][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = blockIdx.x / splits;
    const int64_t lo = min(c, ((int64_t)(blockIdx.x - row * splits) * LP_WAVES + wave) * seg_len), hi = min(c, lo + seg_len);
    const T* x = scores + row * ld;
    const Row r(x, targets, row, c);
    int before = 0;
    Best best(TOP ? pend + wave * ROOM : nullptr, k);
    Stat st = walk<T, ENT, RANK, TOP>(x, lo, hi, c1, r.target, r.score, before, best);
    if (lane == 0) found[wave] = Part{st.m, st.s, st.e, before};
    if constexpr (TOP) lists[wave][lane] = best.list;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 1; w < LP_WAVES; ++w) {
        Stat b;
        b.m = found[w].m, b.s = found[w].s, b.e = found[w].e;
        st = join(st, b, c1);
        before += found[w].before;
        if constexpr (TOP) best.take(lists[w][63 - lane]);
    }
    if (!parts) {
        if (lane == 0) write_row(st, before, row, r.score, r.there, temp, out);
        if constexpr (TOP) write_top(best.list, k, row, st, temp, out);
    } else {
        if (lane == 0) parts[blockIdx.x] = Part{st.m, st.s, st.e, before};
        if constexpr (TOP)
            if (lane < k) keys[(int64_t)blockIdx.x * k + lane] = best.list;
    }
}

// One wave a row: joins the parts of its blocks in their order.
template <class T>
__global__ __launch_bounds__(64) void logprobs_join_kernel(const T* __restrict__ scores, int64_t c, int64_t ld, float c1,
                                                           float temp, const int64_t* __restrict__ targets, int k,
                                                           int splits, const Part* __restrict__ parts,
                                                           const u64* __restrict__ keys, LogProbsOut out) {
    __shared__ u64 pend[Best::ROOM];
    const int lane = threadIdx.x;
    const int64_t row = blockIdx.x;
    const Row r(scores + row * ld, targets, row, c);
    Stat st;
    int before = 0;
    for (int i = lane; i < splits; i += 64) {
        const Part p = parts[row * splits + i];
        Stat b;
        b.m = p.m, b.s = p.s, b.e = p.e;
        st = join(st, b, c1);
        before += p.before;
    }
    st = join_lanes(st, c1);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) before += __shfl_xor(before, o);
    if (lane == 0) write_row(st, before, row, r.score, r.there, temp, out);
    if (k) {
        Best best(pend, k);
        const u64* list = keys + row * splits * k;
        const int total = splits * k;
        // the k-th best of the first 64 parts' best keys bounds the k-th best score
        const u64 first = lane < splits ? list[lane * k] : 0;
        const u64 kth = lane_value(sort_up(first), 64 - k);
        if (kth) best.bound(key_score(kth));
        for (int i = 0; i < total; i += 8 * 64) {
            u64 x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) x[u] = i + u * 64 + lane < total ? list[i + u * 64 + lane] : 0;
            for (int u = 0; u < 8; ++u)
                if (__any(x[u] > best.tau)) {
                    best.offer(x[u], x[u] != 0);
                    best.settle();
                }
        }
        if (best.waiting) best.flush();
        write_top(best.list, k, row, st, temp, out);
    }
}

// ---------------------------------------------------------------- gradient
// ds = p (-g_t - g_H (log p + H)) + [j = t] g_t, over T. Bound by HBM: bf16 8192 x 32000 190 to 199 us, 5.4
// TB/s read and written; f32 2503 x 10007 with entropy 31 to 39 (partly from the cache).
// A wave: U * 64 * N neighbouring elements of one row. All loads go out before the first use (503 us
// for the first without).
template <class T, bool ENT, int U>
__global__ __launch_bounds__(256) void logprobs_backward_kernel(
    const T* scores, int64_t n, int64_t c, int64_t ld, float c1, float inv_t, const int64_t* __restrict__ targets,
    const float* __restrict__ stats, const float* __restrict__ grad_logp, const float* __restrict__ entropy,
    const float* __restrict__ grad_entropy, T* grad, int64_t ld_grad, uint32_t per_row) {
    constexpr int N = Vec16<T>::N;
    const int lane = threadIdx.x & 63;
    const uint32_t w = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t row = w / per_row;
    if (row >= n) return;
    const int64_t at = (int64_t)(w - row * per_row) * (64 * N * U);
    const T* x = scores + row * ld;
    T* g = grad + row * ld_grad;
    Vec16<T> v[U];
    const bool whole = at + 64 * N * U <= c;
    if (whole) {
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = load16(x + at + (u * 64 + lane) * N);
    } else {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t p = at + (u * 64 + lane) * N;
            if (p + N <= c) v[u] = load16(x + p);
            else
#pragma unroll
                for (int j = 0; j < N; ++j) v[u].v[j] = p + j < c ? x[p + j] : (T)0.0f;
        }
    }
    int64_t target = targets ? targets[row] : -1;
    if (target >= c) target = -1;
    float m = stats[2 * (int64_t)row], log_sum2 = stats[2 * (int64_t)row + 1] * LOG2E;
    const bool empty = log_sum2 == -INFINITY;
    const float gl = target >= 0 && grad_logp && !empty ? grad_logp[row] * inv_t : 0.0f;
    const float gh = ENT && !empty ? grad_entropy[row] * inv_t : 0.0f, h = ENT ? entropy[row] : 0.0f;
    if (empty) m = 0.0f, log_sum2 = INFINITY;  // p = 0 everywhere
    const bool has = target >= at && target < at + 64 * N * U;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t p = at + (u * 64 + lane) * N;
        float d[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float lp = fmaf((float)v[u].v[j] - m, c1, -log_sum2), pr = __builtin_amdgcn_exp2f(lp);
            if constexpr (ENT) d[j] = pr * fmaf(-gh, fmaf(fmaxf(lp, FLOOR_U), LN2, h), -gl);
            else d[j] = pr * -gl;
        }
        if (has) {
            const int t = (int)(target - at) - (u * 64 + lane) * N;
#pragma unroll
            for (int j = 0; j < N; ++j) d[j] += j == t ? gl : 0.0f;
        }
        Vec16<T> o;
#pragma unroll
        for (int j = 0; j < N; ++j) o.v[j] = (T)d[j];
        if (whole || p + N <= c) store16(g + p, o);
        else
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (p + j < c) g[p + j] = o.v[j];
    }
}

}  // namespace

void log_probs(int32_t dtype, const void* scores, int64_t n, int64_t c, int64_t ld, float temperature,
               const int64_t* targets, int k, const LogProbsOut& out) {
    const float c1 = (float)(1.44269504088896340736 / (double)temperature);
    with_dtype(dtype, [&](auto zero) {
        using T = decltype(zero);
        constexpr int64_t STEP = Step<T>::SIZE;
        // A row goes to one wave where there are 8 rows a CU, else to a block, and to several where there
        // are fewer rows than CUs, which costs another launch to join them. Best 5, wave and block: f32
        // 3000 x 10007 26 and 30 us, 2048 x 10007 23.0 and 23.5, 1500 x 10007 23 and 18; bf16 4096 x 32000 59
        // and 69, 2048 x 32000 42 and 39. One block and two or more: f32 700 x 10007 12 and 19, 256 x 10007 9.7
        // and 13.5, 64 x 32000 13.9 and 12.4, bf16 150 x 32000 16.5 and 14.9.
        const int cus = device().num_cus;
        const int64_t steps = (c + STEP - 1) / STEP;
        const bool by_wave = n >= 8LL * cus || steps == 1;
        int64_t splits = n >= cus ? 1 : std::min<int64_t>((2LL * cus + n - 1) / n, (steps + LP_WAVES - 1) / LP_WAVES);
        const int64_t seg = (steps + splits * LP_WAVES - 1) / (splits * LP_WAVES) * STEP;
        splits = by_wave ? 1 : (c + seg * LP_WAVES - 1) / (seg * LP_WAVES);
        Part* parts = nullptr;
        u64* keys = nullptr;
        if (splits > 1) {
            parts = (Part*)scratch_bytes("lp_parts", n * splits * (int64_t)sizeof(Part));
            keys = (u64*)scratch_bytes("lp_keys", std::max<int64_t>(1, n * splits * k) * 8);
        }
        const int64_t slice = ((int64_t)1 << 23) / splits;  // rows of one launch: at most 2^31 threads
        for (int64_t r = 0; r < n; r += slice) {
            const int64_t rows = std::min(slice, n - r);
            const T* x = (const T*)scores + r * ld;
            const int64_t* t = targets ? targets + r : nullptr;
            LogProbsOut o = out;
            if (o.logp) o.logp += r;
            if (o.rank) o.rank += r;
            if (o.entropy) o.entropy += r;
            if (o.stats) o.stats += 2 * r;
            if (o.top_ids) o.top_ids += r * k;
            if (o.top_logp) o.top_logp += r * k;
            auto go = [&](auto ent, auto rank, auto top) {
                constexpr bool E = decltype(ent)::value, R = decltype(rank)::value, K = decltype(top)::value;
                if (by_wave)
                    RVX_LAUNCH("log_probs", (logprobs_wave_kernel<T, E, R, K>),
                               dim3((unsigned)((rows + LP_WAVES - 1) / LP_WAVES)), dim3(64 * LP_WAVES), 0, x, rows, c, ld, c1,
                               temperature, t, k, o);
                else
                    RVX_LAUNCH("log_probs", (logprobs_block_kernel<T, E, R, K>), dim3((unsigned)(rows * splits)),
                               dim3(64 * LP_WAVES), 0, x, c, ld, c1, temperature, t, k, (int)splits, seg, parts, keys, o);
            };
            auto flag = [](bool on, auto&& f) {
                if (on) f(std::true_type{});
                else f(std::false_type{});
            };
            flag(out.entropy != nullptr, [&](auto e) {
                flag(out.rank != nullptr, [&](auto q) { flag(k > 0, [&](auto p) { go(e, q, p); }); });
            });
            if (splits > 1)
                RVX_LAUNCH("log_probs_join", logprobs_join_kernel<T>, dim3((unsigned)rows), dim3(64), 0, x, c, ld, c1, temperature, t,
                           k, (int)splits, (const Part*)parts, (const u64*)keys, o);
        }
    });
}

void log_probs_backward(int32_t dtype, const void* scores, int64_t n, int64_t c, int64_t ld, float temperature,
                        const int64_t* targets, const float* stats, const float* grad_logp, const float* entropy,
                        const float* grad_entropy, void* grad, int64_t ld_grad) {
    const float inv_t = (float)(1.0 / (double)temperature), c1 = (float)(1.44269504088896340736 / (double)temperature);
    with_dtype(dtype, [&](auto zero) {
        using T = decltype(zero);
        auto go = [&](auto unroll, auto ent) {
            constexpr int U = decltype(unroll)::value;
            constexpr int64_t CHUNK = 64 * Vec16<T>::N * U;
            const int64_t per_row = (c + CHUNK - 1) / CHUNK;
            const int64_t slice = std::max<int64_t>(1, ((int64_t)1 << 25) / per_row);  // at most 2^31 threads
            for (int64_t r = 0; r < n; r += slice) {
                const int64_t rows = std::min(slice, n - r);
                RVX_LAUNCH("log_probs_backward", (logprobs_backward_kernel<T, decltype(ent)::value, U>),
                           dim3((unsigned)((rows * per_row + 3) / 4)), dim3(256), 0, (const T*)scores + r * ld, rows, c, ld, c1,
                           inv_t, targets ? targets + r : nullptr, stats + 2 * r, grad_logp ? grad_logp + r : nullptr,
                           entropy ? entropy + r : nullptr, grad_entropy ? grad_entropy + r : nullptr,
                           (T*)grad + r * ld_grad, ld_grad, (uint32_t)per_row);
            }
        };
        auto by_width = [&](auto ent) {
            // U 4 and 1: f32 8192 x 1000 11.7 and 14.0 us; bf16 8192 x 3000 22.4 and 22.7, 8192 x 1000 12.7 and 8.5
            if (c > 64 * Vec16<T>::N * 2) go(std::integral_constant<int, 4>{}, ent);
            else go(std::integral_constant<int, 1>{}, ent);
        };
        if (grad_entropy) by_width(std::true_type{});
        else by_width(std::false_type{});
    });
}

}  // namespace rvx
