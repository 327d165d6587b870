// k_logprobs.hip — log probabilities of given ids over rows of scores, with rank, entropy and
// the best alternatives, in one pass over the scores; and the gradient by the scores.
//
// With u = (s - m) / T, m the row's largest score, S = sum e^u and E = sum e^u u:
//   log p_t = u_t - ln S,   H = -sum p ln p = ln S - E / S.
// m, S and E over a part of a row join with those over another part (m' = max, S' = S r + ..,
// E' = r (E + S d) + .. with d = (m - m') / T, r = e^d), so one pass suffices. All three are
// kept in 32 bits, in units of log2, for v_exp_f32.
#include "heads.hpp"

namespace rvx {
namespace {

constexpr float LN2 = 0.69314718055994530942f, LOG2E = 1.44269504088896340736f;
constexpr float FLOOR_U = -1e30f;  // e^u is 0 long before; keeps 0 * u finite for masked scores
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

// The 64 best keys a wave has seen, one a lane, best first. Keys above the k-th best wait in LDS;
// 64 of them at a time are sorted (bitonic, ascending) and merged: max(best, new) of a descending and
// an ascending row holds the 64 largest as a bitonic row.
struct Best {
    u64 list = 0, tau = 0;  // tau: the k-th best key
    float tau_score = -INFINITY;
    int waiting = 0, k;
    u64* pend;  // this wave's waiting keys: room for 64 and for what is offered between two flushes
    __device__ Best(u64* p, int kk) : k(kk), pend(p) {}

    __device__ void merge(u64 x) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int size = 2; size <= 64; size <<= 1)
#pragma unroll
            for (int st = size >> 1; st > 0; st >>= 1) {
                const u64 y = __shfl_xor(x, st);
                const bool up = (lane & size) == 0, low = (lane & st) == 0;
                x = (low == up) == (x < y) ? x : y;
            }
        u64 z = list > x ? list : x;
#pragma unroll
        for (int st = 32; st > 0; st >>= 1) {
            const u64 y = __shfl_xor(z, st);
            z = ((lane & st) == 0) == (z > y) ? z : y;
        }
        list = z;
        tau = __shfl(list, k - 1);
        tau_score = tau ? key_score(tau) : -INFINITY;
    }
    __device__ void flush() {  // the last 64 waiting keys
        const int lane = threadIdx.x & 63;
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "workgroup");
        const int from = max(0, waiting - 64);
        const u64 x = from + lane < waiting ? pend[from + lane] : 0;
        waiting = from;
        if (__any(x > tau)) merge(x);
    }
    __device__ __forceinline__ void offer(u64 key, bool there) {
        const bool in = there && key > tau;
        const u64 mask = __ballot(in);
        if (in)
            pend[waiting + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                                     __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0))] = key;
        waiting += __popcll(mask);
    }
};

struct Part {  // what one wave found of one row
    float m, s, e;
    int before;
};

__device__ __forceinline__ void write_row(const Stat& st, int before, int64_t row, float st_score, bool has_target,
                                          float inv_t, const LogProbsOut& out) {
    const bool empty = st.s == 0.0f;
    const float m = empty ? -INFINITY : st.m;
    const float log_sum = empty ? -INFINITY : logf(st.s);
    if (out.logp) out.logp[row] = !has_target ? 0.0f : empty ? -INFINITY : (st_score - m) * inv_t - log_sum;
    if (out.rank) out.rank[row] = has_target ? before : -1;
    if (out.entropy) out.entropy[row] = empty ? 0.0f : log_sum - LN2 * (st.e / st.s);
    if (out.stats) {
        out.stats[2 * row] = m;
        out.stats[2 * row + 1] = log_sum;
    }
}
__device__ __forceinline__ void write_top(u64 list, int k, int64_t row, const Stat& st, float inv_t,
                                          const LogProbsOut& out) {
    const int lane = threadIdx.x & 63;
    if (lane >= k) return;
    const bool none = list == 0;
    if (out.top_ids) out.top_ids[row * k + lane] = none ? -1 : (int64_t)(0xffffffffu - (uint32_t)list);
    if (out.top_logp)
        out.top_logp[row * k + lane] = none ? -INFINITY : (key_score(list) - st.m) * inv_t - logf(st.s);
}

constexpr int LP_U = 2, LP_WAVES = 4;  // 16-byte loads per lane and step; waves per block

// One wave: elements [seg * seg_len, ..) of one row. parts == null: the wave has the whole row.
template <class T, bool ENT, bool RANK, bool TOP>
__global__ __launch_bounds__(64 * LP_WAVES) void logprobs_kernel(const T* __restrict__ scores, int64_t n, int64_t c,
                                                                int64_t ld, float c1, float inv_t,
                                                                const int64_t* __restrict__ targets, int k,
                                                                int splits, int64_t seg_len, Part* parts, u64* keys,
                                                                LogProbsOut out) {
    constexpr int N = Vec16<T>::N, STEP = 64 * N * LP_U;
    constexpr int ROOM = 64 + 64 * N;
    __shared__ u64 pend[TOP ? LP_WAVES * ROOM : 1];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t w = (int64_t)blockIdx.x * LP_WAVES + wave;
    if (w >= n * splits) return;
    const int64_t row = w / splits;
    const int64_t lo = (w - row * splits) * seg_len, hi = min(c, lo + seg_len);
    const T* x = scores + row * ld;
    int64_t target = targets ? targets[row] : -1;
    const bool has_target = target >= 0 && target < c;
    const float st_score = has_target ? (float)x[target] : NAN;
    if (!has_target) target = -1;

    Stat st;
    int before = 0;
    Best best(TOP ? pend + wave * ROOM : nullptr, k);
    for (int64_t at = lo; at < hi; at += STEP) {
        float v[LP_U][N];
        const bool whole = at + STEP <= hi;
#pragma unroll
        for (int u = 0; u < LP_U; ++u) {
            const int64_t p = at + (u * 64 + lane) * N;
            if (whole || p + N <= hi) {
                const Vec16<T> r = load16(x + p);
#pragma unroll
                for (int j = 0; j < N; ++j) v[u][j] = (float)r.v[j];
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j) v[u][j] = p + j < hi ? (float)x[p + j] : -INFINITY;
            }
        }
        float cm = -INFINITY;
#pragma unroll
        for (int u = 0; u < LP_U; ++u)
#pragma unroll
            for (int j = 0; j < N; ++j) cm = fmaxf(cm, v[u][j]);
        {
            const float mn = fmaxf(st.m, cm);
            const float d = fmaxf((st.m - mn) * c1, FLOOR_U), r = __builtin_amdgcn_exp2f(d);
            float s = 0.f, e = 0.f;
#pragma unroll
            for (int u = 0; u < LP_U; ++u)
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const float y = (v[u][j] - mn) * c1, ex = __builtin_amdgcn_exp2f(y);
                    s += ex;
                    if constexpr (ENT) e = fmaf(ex, fmaxf(y, FLOOR_U), e);
                }
            if constexpr (ENT) st.e = fmaf(r, fmaf(st.s, d, st.e), e);
            st.s = fmaf(st.s, r, s);
            st.m = mn;
        }
        if constexpr (RANK) {
            if (at + STEP <= target) {
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
#pragma unroll
                for (int u = 0; u < LP_U; ++u)
#pragma unroll
                    for (int j = 0; j < N; ++j)
                        before += __popcll(__ballot(
                            v[u][j] > st_score || (v[u][j] == st_score && at + (u * 64 + lane) * N + j < target)));
            }
        }
        if constexpr (TOP) {
            if (__any(cm > best.tau_score)) {
#pragma unroll
                for (int u = 0; u < LP_U; ++u) {
#pragma unroll
                    for (int j = 0; j < N; ++j)
                        best.offer(key_of(v[u][j], (uint32_t)(at + (u * 64 + lane) * N + j)), v[u][j] > -INFINITY);
                    while (best.waiting >= 64) best.flush();
                }
            }
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        Stat b;
        b.m = __shfl_xor(st.m, o), b.s = __shfl_xor(st.s, o), b.e = __shfl_xor(st.e, o);
        st = join(st, b, c1);
    }
    if constexpr (TOP)
        if (best.waiting) best.flush();
    if (!parts) {
        if (lane == 0) write_row(st, before, row, st_score, has_target, inv_t, out);
        if constexpr (TOP) write_top(best.list, k, row, st, inv_t, out);
    } else {
        if (lane == 0) parts[w] = Part{st.m, st.s, st.e, before};
        if constexpr (TOP)
            if (lane < k) keys[w * k + lane] = best.list;
    }
}

// One wave a row: joins the parts of its splits in their order.
template <class T>
__global__ __launch_bounds__(64) void logprobs_join_kernel(const T* __restrict__ scores, int64_t c, int64_t ld, float c1,
                                                           float inv_t, const int64_t* __restrict__ targets, int k,
                                                           int splits, const Part* __restrict__ parts,
                                                           const u64* __restrict__ keys, LogProbsOut out) {
    __shared__ u64 pend[128];
    const int lane = threadIdx.x;
    const int64_t row = blockIdx.x;
    int64_t target = targets ? targets[row] : -1;
    const bool has_target = target >= 0 && target < c;
    const float st_score = has_target ? (float)scores[row * ld + target] : NAN;
    Stat st;
    int before = 0;
    for (int i = lane; i < splits; i += 64) {
        const Part p = parts[row * splits + i];
        Stat b;
        b.m = p.m, b.s = p.s, b.e = p.e;
        st = join(st, b, c1);
        before += p.before;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        Stat b;
        b.m = __shfl_xor(st.m, o), b.s = __shfl_xor(st.s, o), b.e = __shfl_xor(st.e, o);
        st = join(st, b, c1);
        before += __shfl_xor(before, o);
    }
    if (lane == 0) write_row(st, before, row, st_score, has_target, inv_t, out);
    if (k) {
        Best best(pend, k);
        for (int i = 0; i < splits * k; i += 64) {
            const u64 key = i + lane < splits * k ? keys[row * splits * k + i + lane] : 0;
            best.offer(key, key != 0);
            while (best.waiting >= 64) best.flush();
        }
        if (best.waiting) best.flush();
        write_top(best.list, k, row, st, inv_t, out);
    }
}

constexpr int LB_U = 2;  // 16-byte loads per lane

template <class T, bool ENT>
__global__ __launch_bounds__(256) void logprobs_backward_kernel(
    const T* scores, int64_t c, int64_t ld, float c1, float inv_t, const int64_t* __restrict__ targets,
    const float* __restrict__ stats, const float* __restrict__ grad_logp, const float* __restrict__ entropy,
    const float* __restrict__ grad_entropy, T* grad, int64_t ld_grad, int blocks_per_row) {
    constexpr int N = Vec16<T>::N;
    const int64_t row = blockIdx.x / blocks_per_row;
    const int64_t at = (int64_t)(blockIdx.x - row * blocks_per_row) * (256 * N * LB_U);
    int64_t target = targets ? targets[row] : -1;
    const bool has_target = target >= 0 && target < c;
    const float m = stats[2 * row], log_sum = stats[2 * row + 1], log_sum2 = log_sum * LOG2E;
    const bool empty = log_sum == -INFINITY;
    const float gl = has_target && grad_logp && !empty ? grad_logp[row] * inv_t : 0.0f;
    const float gh = ENT ? grad_entropy[row] * inv_t : 0.0f, h = ENT ? entropy[row] : 0.0f;
    if (!has_target) target = -1;
#pragma unroll
    for (int u = 0; u < LB_U; ++u) {
        const int64_t p = at + (u * 256 + threadIdx.x) * N;
        if (p >= c) return;
        const T* x = scores + row * ld + p;
        T* g = grad + row * ld_grad + p;
        const bool whole = p + N <= c;
        Vec16<T> v;
        if (whole) v = load16(x);
        else
            for (int j = 0; j < N; ++j) v.v[j] = p + j < c ? x[j] : (T)0.0f;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float lp = fmaf((float)v.v[j] - m, c1, -log_sum2), pr = __builtin_amdgcn_exp2f(lp);
            float d = -gl * pr;
            if constexpr (ENT) d = fmaf(-gh * pr, fmaf(fmaxf(lp, FLOOR_U), LN2, h), d);
            if (empty) d = 0.0f;
            if (p + j == target) d += gl;
            v.v[j] = (T)d;
        }
        if (whole) store16(g, v);
        else
            for (int j = 0; j < N; ++j)
                if (p + j < c) g[j] = v.v[j];
    }
}

}  // namespace

void log_probs(int32_t dtype, const void* scores, int64_t n, int64_t c, int64_t ld, float temperature,
               const int64_t* targets, int k, const LogProbsOut& out) {
    const float inv_t = (float)(1.0 / (double)temperature), c1 = (float)(1.44269504088896340736 / (double)temperature);
    with_dtype(dtype, [&](auto zero) {
        using T = decltype(zero);
        constexpr int64_t STEP = 64 * Vec16<T>::N * LP_U;
        // A row goes to one wave unless that leaves CUs without work: 16 waves a CU hide the loads.
        const int64_t want = (16LL * device().num_cus + n - 1) / n, most = (c + STEP - 1) / STEP;
        int64_t splits = std::max<int64_t>(1, std::min(want, most));
        const int64_t seg = ((most + splits - 1) / splits) * STEP;
        splits = (c + seg - 1) / seg;
        Part* parts = nullptr;
        u64* keys = nullptr;
        if (splits > 1) {
            parts = (Part*)scratch_bytes("lp_parts", n * splits * (int64_t)sizeof(Part));
            keys = (u64*)scratch_bytes("lp_keys", std::max<int64_t>(1, n * splits * k) * 8);
        }
        const bool ent = out.entropy != nullptr, rank = out.rank != nullptr, top = k > 0;
        const int64_t slice = ((int64_t)1 << 25) / splits;  // rows of one launch: at most 2^31 threads
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
        const dim3 grid((unsigned)((rows * splits + LP_WAVES - 1) / LP_WAVES));
        auto go = [&](auto kernel) {
            RVX_LAUNCH("log_probs", kernel, grid, dim3(64 * LP_WAVES), 0, x, rows, c, ld, c1, inv_t, t, k, (int)splits,
                       seg, parts, keys, o);
        };
        if (ent && rank && top) go(logprobs_kernel<T, true, true, true>);
        else if (ent && rank) go(logprobs_kernel<T, true, true, false>);
        else if (ent && top) go(logprobs_kernel<T, true, false, true>);
        else if (ent) go(logprobs_kernel<T, true, false, false>);
        else if (rank && top) go(logprobs_kernel<T, false, true, true>);
        else if (rank) go(logprobs_kernel<T, false, true, false>);
        else if (top) go(logprobs_kernel<T, false, false, true>);
        else go(logprobs_kernel<T, false, false, false>);
        if (splits > 1)
            RVX_LAUNCH("log_probs_join", logprobs_join_kernel<T>, dim3((unsigned)rows), dim3(64), 0, x, c, ld, c1, inv_t, t,
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
        constexpr int64_t BLOCK = 256 * Vec16<T>::N * LB_U;
        const int64_t per_row = (c + BLOCK - 1) / BLOCK;
        // rows go in slices of at most 2^31 threads
        const int64_t slice = std::max<int64_t>(1, ((int64_t)1 << 23) / per_row);
        for (int64_t r = 0; r < n; r += slice) {
            const dim3 grid((unsigned)(std::min(slice, n - r) * per_row));
            auto go = [&](auto kernel) {
                RVX_LAUNCH("log_probs_backward", kernel, grid, dim3(256), 0, (const T*)scores + r * ld, c, ld, c1, inv_t,
                           targets ? targets + r : nullptr, stats + 2 * r, grad_logp ? grad_logp + r : nullptr,
                           entropy ? entropy + r : nullptr, grad_entropy ? grad_entropy + r : nullptr,
                           (T*)grad + r * ld_grad, ld_grad, (int)per_row);
            };
            if (grad_entropy) go(logprobs_backward_kernel<T, true>);
            else go(logprobs_backward_kernel<T, false>);
        }
    });
}

}  // namespace rvx
