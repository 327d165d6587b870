// k_embedding.hip — rows of a learned table by id, and the gradient of the table.
//
// Forward: out[i] = scale * table[id_i]; one read and one write of each row, bound by HBM.
// Backward: g[v] = scale * sum_{i: id_i = v} dy[i]. The positions are grouped by id with a stable
// radix sort of (id, i), so a row's sum runs over i in ascending order whatever ran when: no
// floating-point atomics, the same bits every call.
#include "heads.hpp"

namespace rvx {
namespace {

// ---------------------------------------------------------------- forward
constexpr int EF_U = 4;  // 16-byte chunks per lane

template <class T>
__global__ __launch_bounds__(256) void embed_forward_kernel(const T* __restrict__ table, int64_t rows, int dim, int cpr,
                                                           uint32_t inv_cpr, const int64_t* __restrict__ ids, int64_t n,
                                                           float scale, T* __restrict__ out) {
    constexpr int N = Vec16<T>::N;
    const int64_t first = (int64_t)blockIdx.x * (256 * EF_U);
    const int64_t row0 = first / cpr;
    const uint32_t rem0 = (uint32_t)(first - row0 * cpr);
    int64_t id[EF_U];
    int64_t row[EF_U];
    uint32_t col[EF_U];
#pragma unroll
    for (int u = 0; u < EF_U; ++u) {
        const uint32_t x = rem0 + u * 256 + threadIdx.x;
        const uint32_t q = cpr == 1 ? x : __umulhi(x, inv_cpr);  // x / cpr: exact for x * cpr < 2^32
        row[u] = row0 + q;
        col[u] = (x - q * cpr) * N;
        id[u] = row[u] < n ? ids[row[u]] : -1;
    }
    Vec16<T> v[EF_U];
#pragma unroll
    for (int u = 0; u < EF_U; ++u) {
        const bool there = id[u] >= 0 && id[u] < rows;
        const T* p = table + id[u] * dim + col[u];
        if (there && col[u] + N <= (uint32_t)dim) v[u] = load16(p);
        else
#pragma unroll
            for (int j = 0; j < N; ++j) v[u].v[j] = there && col[u] + j < (uint32_t)dim ? p[j] : (T)0.0f;
    }
#pragma unroll
    for (int u = 0; u < EF_U; ++u) {
        if (row[u] >= n) continue;
        Vec16<T> r;
#pragma unroll
        for (int j = 0; j < N; ++j) r.v[j] = (T)((float)v[u].v[j] * scale);
        T* o = out + row[u] * dim + col[u];
        if (col[u] + N <= (uint32_t)dim) store16(o, r);
        else
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (col[u] + j < (uint32_t)dim) o[j] = r.v[j];
    }
}

// ---------------------------------------------------------------- grouping positions by id
// Stable LSD radix sort of (key, position), key = id, or `rows` for an absent id. The n positions
// are cut into at most SORT_TILES tiles, one block each. A pass is two launches: every tile counts
// its digits in LDS, then moves its elements; for that each block sums the counts of the tiles
// before it by itself, which costs less than a launch for a scan.
constexpr int SORT_TILES = 64, SORT_THREADS = 512, SORT_WAVES = SORT_THREADS / 64, SORT_STEP = SORT_THREADS * 4;
constexpr int SORT_MAX_BITS = 11, SORT_BINS = 1 << SORT_MAX_BITS;

__device__ __forceinline__ uint32_t sort_key(const int64_t* ids, int64_t i, uint32_t rows) {
    const int64_t id = ids[i];
    return id >= 0 && id < (int64_t)rows ? (uint32_t)id : rows;
}

template <bool FIRST>
__global__ __launch_bounds__(SORT_THREADS) void sort_count_kernel(const int64_t* __restrict__ ids,
                                                                 const uint32_t* __restrict__ key_in, int64_t n,
                                                                 uint32_t rows, int64_t tile, int bits, int shift,
                                                                 uint32_t* __restrict__ counts) {
    __shared__ uint32_t hist[SORT_BINS];
    const int bins = 1 << bits;
    for (int d = threadIdx.x; d < bins; d += SORT_THREADS) hist[d] = 0;
    __syncthreads();
    const int64_t lo = blockIdx.x * tile, hi = min(n, lo + tile);
#pragma unroll 4
    for (int64_t i = lo + threadIdx.x; i < hi; i += SORT_THREADS) {
        const uint32_t key = FIRST ? sort_key(ids, i, rows) : key_in[i];
        atomicAdd(&hist[(key >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < bins; d += SORT_THREADS) counts[((int64_t)blockIdx.x << bits) | d] = hist[d];
}

// FIRST: the elements are ids in their own order; else (key, pos) of the pass before.
template <bool FIRST>
__global__ __launch_bounds__(SORT_THREADS) void sort_move_kernel(const int64_t* __restrict__ ids,
                                                                const uint32_t* __restrict__ key_in,
                                                                const uint32_t* __restrict__ pos_in, int64_t n,
                                                                uint32_t rows, int64_t tile, int tiles, int bits,
                                                                int shift, const uint32_t* __restrict__ counts,
                                                                uint32_t* __restrict__ key_out,
                                                                uint32_t* __restrict__ pos_out) {
    __shared__ uint32_t base[SORT_BINS];               // where this block's next element of a digit goes
    __shared__ uint32_t mine[SORT_WAVES][SORT_BINS];   // per wave: its count of a digit, then its next place
    __shared__ uint32_t sums[SORT_THREADS];
    const int bins = 1 << bits, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int me = blockIdx.x;
    // base[d] = elements of smaller digits anywhere + of digit d in the tiles before
    constexpr int PER = SORT_BINS / SORT_THREADS;
    uint32_t total[PER], ahead[PER], sum = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int d = t * PER + j;
        total[j] = ahead[j] = 0;
        if (d < bins)
#pragma unroll 8
            for (int b = 0; b < tiles; ++b) {
                const uint32_t v = counts[(int64_t)b << bits | d];
                total[j] += v;
                ahead[j] += b < me ? v : 0;
            }
        sum += total[j];
    }
    sums[t] = sum;
    __syncthreads();
    for (int o = 1; o < SORT_THREADS; o <<= 1) {
        const uint32_t v = t >= o ? sums[t - o] : 0;
        __syncthreads();
        sums[t] += v;
        __syncthreads();
    }
    uint32_t run = t ? sums[t - 1] : 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        base[t * PER + j] = run + ahead[j];
        run += total[j];
    }
    const int64_t lo = me * tile, hi = min(n, lo + tile);
    for (int64_t at = lo; at < hi; at += SORT_STEP) {
        __syncthreads();
        for (int d = t; d < bins; d += SORT_THREADS)
            for (int w = 0; w < SORT_WAVES; ++w) mine[w][d] = 0;
        __syncthreads();
        // a wave has 4 x 64 elements in order
        uint32_t key[4], pos[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t i = at + wave * 256 + u * 64 + lane;
            key[u] = 0xffffffffu;
            pos[u] = 0;
            if (i < hi) {
                key[u] = FIRST ? sort_key(ids, i, rows) : key_in[i];
                pos[u] = FIRST ? (uint32_t)i : pos_in[i];
                atomicAdd(&mine[wave][(key[u] >> shift) & (bins - 1)], 1u);
            }
        }
        __syncthreads();
        for (int d = t; d < bins; d += SORT_THREADS) {
            uint32_t b = base[d];
            for (int w = 0; w < SORT_WAVES; ++w) {
                const uint32_t v = mine[w][d];
                mine[w][d] = b;
                b += v;
            }
            base[d] = b;
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const bool there = at + wave * 256 + u * 64 + lane < hi;
            const uint32_t d = (key[u] >> shift) & (bins - 1);
            unsigned long long same = __ballot(there);
            for (int b = 0; b < bits; ++b) {
                const unsigned long long m = __ballot((d >> b) & 1);
                same &= (d >> b) & 1 ? m : ~m;
            }
            const int before = __popcll(same & ((1ull << lane) - 1));
            uint32_t to = 0;
            if (there) to = mine[wave][d] + before;
            __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "workgroup");
            if (there && before == 0) mine[wave][d] = to + __popcll(same);
            __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "workgroup");
            if (there) {
                key_out[to] = key[u];
                pos_out[to] = pos[u];
            }
        }
    }
}

// ---------------------------------------------------------------- sums over groups
// A long group is summed in two steps: GROUP neighbouring entries of the sorted order that share
// one id are first summed to a partial row (level 1), GROUP such partial rows to another (level
// 2), each by a wave of its own; the row's wave then adds partial rows. What is a group depends
// on the sorted ids alone, and so does the order of the additions.
constexpr int GROUP = 64;

template <class T>
struct Slab {  // a wave's columns of a row: N a lane
    static constexpr int N = Vec16<T>::N, COLS = 64 * N;
};

// acc += columns [col, col + N) of `count` (<= 64) rows; row j's start is row_of(j), wave-uniform
template <class S, int N, class F>
__device__ __forceinline__ void add_rows(float (&acc)[N], int count, int col, int dim, F&& row_of) {
    constexpr int U = 4;
    static_assert(N % Vec16<S>::N == 0, "a lane's columns are whole vectors");
    for (int j = 0; j < count; j += U) {
        S v[U][N];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (j + u < count) {
                const S* p = row_of(j + u) + col;
                if (col + N <= dim) {
                    __builtin_memcpy(v[u], p, sizeof(S) * N);
                } else {
#pragma unroll
                    for (int i = 0; i < N; ++i) v[u][i] = col + i < dim ? p[i] : (S)0.0f;
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (j + u < count)
#pragma unroll
                for (int i = 0; i < N; ++i) acc[i] += (float)v[u][i];
    }
}

// level 1 (SRC = T, rows by position) and level 2 (SRC = float, rows in their order): partial rows
template <class T, bool SECOND>
__global__ __launch_bounds__(256) void embed_partial_kernel(const T* __restrict__ grad_out,
                                                           const float* __restrict__ first, int dim,
                                                           const uint32_t* __restrict__ key,
                                                           const uint32_t* __restrict__ pos, int64_t groups,
                                                           uint32_t rows, float* __restrict__ out) {
    constexpr int N = Slab<T>::N;
    const int lane = threadIdx.x & 63;
    const int64_t g = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (g >= groups) return;
    constexpr int64_t SPAN = SECOND ? GROUP * GROUP : GROUP;
    const uint32_t k = key[g * SPAN];
    if (k >= rows || key[g * SPAN + SPAN - 1] != k) return;
    const int col = blockIdx.y * Slab<T>::COLS + lane * N;
    if (col >= dim) return;
    float acc[N] = {};
    if constexpr (SECOND) {
        add_rows<float>(acc, GROUP, col, dim, [&](int j) { return first + (g * GROUP + j) * dim; });
    } else {
        const uint32_t* p = pos + g * SPAN;
        add_rows<T>(acc, GROUP, col, dim, [&](int j) { return grad_out + (int64_t)p[j] * dim; });
    }
    float* o = out + g * dim + col;
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (col + i < dim) o[i] = acc[i];
}

// columns [col, col + N) of a row that is added to (read early: the load does not wait for the sum)
template <class S, int N>
__device__ __forceinline__ void get_row(const S* o, S (&v)[N], int col, int dim) {
    if (col + N <= dim) __builtin_memcpy(v, o, sizeof(v));
    else
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = col + i < dim ? o[i] : (S)0.0f;
}
template <class S, int N, bool ADD>
__device__ __forceinline__ void put_row(S* o, const float (&acc)[N], S (&v)[N], int col, int dim, float scale) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (S)(ADD ? fmaf(acc[i], scale, (float)v[i]) : acc[i] * scale);
    if (col + N <= dim) __builtin_memcpy(o, v, sizeof(v));
    else
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (col + i < dim) o[i] = v[i];
}

// One wave per (sorted entry, slab): the first entry of an id sums the id's rows.
template <class T, class S, bool ADD>
__global__ __launch_bounds__(256) void embed_rows_kernel(const T* __restrict__ grad_out, int dim, int64_t begin,
                                                        const uint32_t* __restrict__ key,
                                                        const uint32_t* __restrict__ pos, int64_t n, uint32_t rows,
                                                        const float* __restrict__ first,
                                                        const float* __restrict__ second, float scale, S* grad_table) {
    constexpr int N = Slab<T>::N;
    const int lane = threadIdx.x & 63;
    const int64_t i0 = begin + (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (i0 >= n) return;
    // one load gives the entry before, this one and the 62 after it
    const int64_t near_i = i0 + lane - 1;
    const uint32_t near_key = near_i >= 0 && near_i < n ? key[near_i] : 0xffffffffu;  // no key is that large
    const uint32_t near_pos = near_i >= 0 && near_i < n ? pos[near_i] : 0;
    const uint32_t k = __builtin_amdgcn_readlane(near_key, 1);
    if (k >= rows || (uint32_t)__builtin_amdgcn_readlane(near_key, 0) == k) return;
    const int col = blockIdx.y * Slab<T>::COLS + lane * N;
    S* const row = grad_table + (int64_t)k * dim + col;
    S old[N];
    if constexpr (ADD)
        if (col < dim) get_row<S, N>(row, old, col, dim);
    float acc[N] = {};
    const int run = __ffsll(__ballot(lane > 0 && near_key != k) | 1ull << 63) - 2;  // entries of the id, if below 62
    if (run < 62) {
        add_rows<T>(acc, run, min(col, dim), dim,
                    [&](int j) { return grad_out + (int64_t)(uint32_t)__builtin_amdgcn_readlane(near_pos, j + 1) * dim; });
        if (col < dim) put_row<S, N, ADD>(row, acc, old, col, dim, scale);
        return;
    }
    int64_t at = i0;
    while (at < n) {
        if ((at & (GROUP * GROUP - 1)) == 0 && at + GROUP * GROUP <= n && key[at + GROUP * GROUP - 1] == k) {
            const int64_t g = at / (GROUP * GROUP);
            const int64_t left = (n - at) / (GROUP * GROUP);
            const bool same = lane < left && key[at + (int64_t)(lane + 1) * GROUP * GROUP - 1] == k;
            const int count = __ffsll(~__ballot(same)) - 1;
            const int c = count < 0 ? 64 : count;
            if (col < dim) add_rows<float>(acc, c, col, dim, [&](int j) { return second + (g + j) * dim; });
            at += (int64_t)c * GROUP * GROUP;
        } else if ((at & (GROUP - 1)) == 0 && at + GROUP <= n && key[at + GROUP - 1] == k) {
            // partial rows up to the next whole second-level group
            const int64_t g = at / GROUP;
            const int64_t left = min((n - at) / GROUP, (int64_t)GROUP - (g & (GROUP - 1)));
            const bool same = lane < left && key[at + (int64_t)(lane + 1) * GROUP - 1] == k;
            const int count = __ffsll(~__ballot(same)) - 1;
            const int c = count < 0 ? 64 : count;
            if (col < dim) add_rows<float>(acc, c, col, dim, [&](int j) { return first + (g + j) * dim; });
            at += (int64_t)c * GROUP;
        } else {
            // single rows up to the next whole group
            const int left = (int)min(n - at, (int64_t)GROUP - (at & (GROUP - 1)));
            const bool same = lane < left && key[at + lane] == k;
            const int count = __ffsll(~__ballot(same)) - 1;
            const int c = count < 0 ? 64 : count;
            const uint32_t p = same ? pos[at + lane] : 0;
            add_rows<T>(acc, c, min(col, dim), dim,
                        [&](int j) { return grad_out + (int64_t)(uint32_t)__builtin_amdgcn_readlane(p, j) * dim; });
            at += c;
            if (c < left) break;
            continue;
        }
        if (at < n && key[at] != k) break;
    }
    if (col < dim) put_row<S, N, ADD>(row, acc, old, col, dim, scale);
}

// Few positions: no sort. The wave of position i looks for its id among the positions before it
// (then another wave has the row) and adds the rows of the positions after it, in order.
constexpr int SCAN_MAX = 1024;

template <class T, class S, bool ADD>
__global__ __launch_bounds__(256) void embed_scan_kernel(const T* __restrict__ grad_out, int dim,
                                                        const int64_t* __restrict__ ids, int n, int64_t rows,
                                                        float scale, S* grad_table) {
    constexpr int N = Slab<T>::N;
    const int lane = threadIdx.x & 63;
    const int i0 = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (i0 >= n) return;
    const int64_t id = ids[i0];
    if (id < 0 || id >= rows) return;
    for (int j = 0; j < i0; j += 64)
        if (__any(j + lane < i0 && ids[j + lane] == id)) return;
    const int col = blockIdx.y * Slab<T>::COLS + lane * N;
    float acc[N] = {};
    for (int j = i0; j < n; j += 64) {
        unsigned long long m = __ballot(j + lane < n && ids[j + lane] == id);
        const int count = __popcll(m);
        // lane r holds the r-th position of the group's rows
        int mine = 0;
        for (int r = 0; r < count; ++r) {
            const int b = __ffsll(m) - 1;
            m &= m - 1;
            if (lane == r) mine = j + b;
        }
        add_rows<T>(acc, count, min(col, dim), dim,
                    [&](int r) { return grad_out + (int64_t)__builtin_amdgcn_readlane(mine, r) * dim; });
    }
    if (col < dim) {
        S* const row = grad_table + id * dim + col;
        S old[N];
        if constexpr (ADD) get_row<S, N>(row, old, col, dim);
        put_row<S, N, ADD>(row, acc, old, col, dim, scale);
    }
}

__global__ __launch_bounds__(256) void clear_bits_kernel(uint32_t* p, int64_t words) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) p[i] = 0;
}
// a bit for each row that is looked up, from the first entry of each id in the sorted order
__global__ __launch_bounds__(256) void mark_rows_kernel(const uint32_t* __restrict__ key, int64_t n, uint32_t rows,
                                                       uint32_t* present) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const uint32_t k = key[i];
        if (k < rows && (i == 0 || key[i - 1] != k)) atomicOr(&present[k >> 5], 1u << (k & 31));
    }
}

// Rows without an id are zeros: present == null, every row; else the rows whose bit is not set.
__global__ __launch_bounds__(256) void embed_zero_kernel(unsigned char* table, int64_t rows, int64_t row_bytes,
                                                        const uint32_t* __restrict__ present) {
    const int lane = threadIdx.x & 63;
    const int64_t waves = (int64_t)gridDim.x * 4;
    for (int64_t v = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); v < rows; v += waves) {
        if (present && (present[v >> 5] >> (v & 31) & 1)) continue;
        unsigned char* p = table + v * row_bytes;
        const uint4 z = {0, 0, 0, 0};
        int64_t b = (int64_t)lane * 16;
        for (; b + 16 <= row_bytes; b += 64 * 16) __builtin_memcpy(p + b, &z, 16);
        if (b < row_bytes)
            for (; b < row_bytes; b += 2) *(uint16_t*)(p + b) = 0;
    }
}

}  // namespace

void embedding_forward(int32_t dtype, const void* table, int64_t rows, int dim, const int64_t* ids, int64_t n,
                       float scale, void* out) {
    with_dtype(dtype, [&](auto zero) {
        using T = decltype(zero);
        const int cpr = (dim + Vec16<T>::N - 1) / Vec16<T>::N;
        const uint32_t inv = cpr == 1 ? 0 : (uint32_t)((((uint64_t)1 << 32) + cpr - 1) / cpr);
        // launches of at most 2^31 threads
        const int64_t slice = std::max<int64_t>(1, (((int64_t)1 << 31) - 2048) * EF_U / cpr);
        for (int64_t r = 0; r < n; r += slice) {
            const int64_t m = std::min(slice, n - r);
            const int64_t blocks = (m * cpr + 256 * EF_U - 1) / (256 * EF_U);
            RVX_LAUNCH("embedding_forward", embed_forward_kernel<T>, dim3((unsigned)blocks), dim3(256), 0,
                       (const T*)table, rows, dim, cpr, inv, ids + r, m, scale, (T*)out + r * dim);
        }
    });
}

void embedding_backward(int32_t dtype, const void* grad_out, const int64_t* ids, int64_t n, int64_t rows, int dim,
                        float scale, bool accumulate, int32_t table_dtype, void* grad_table) {
    const int64_t row_bytes = (int64_t)dim * dtype_size(table_dtype);
    auto zero_rows = [&](const uint32_t* present) {
        const int64_t blocks = std::min<int64_t>((rows + 3) / 4, 16LL * device().num_cus);
        RVX_LAUNCH("embedding_zero", embed_zero_kernel, dim3((unsigned)blocks), dim3(256), 0, (unsigned char*)grad_table,
                   rows, row_bytes, present);
    };
    auto typed = [&](auto&& f) {  // f(T, S, ADD) of the gradient's, the table's type and the mode
        with_dtype(dtype, [&](auto t) {
            with_dtype(table_dtype, [&](auto s) {
                if (accumulate) f(t, s, std::true_type{});
                else f(t, s, std::false_type{});
            });
        });
    };
    if (n <= SCAN_MAX) {
        if (!accumulate) zero_rows(nullptr);
        if (n == 0) return;
        typed([&](auto t, auto s, auto add) {
            using T = decltype(t);
            using S = decltype(s);
            const int slabs = (dim + Slab<T>::COLS - 1) / Slab<T>::COLS;
            RVX_LAUNCH("embedding_backward", (embed_scan_kernel<T, S, decltype(add)::value>),
                       dim3((unsigned)((n + 3) / 4), slabs), dim3(256), 0, (const T*)grad_out, dim, ids, (int)n,
                       rows, scale, (S*)grad_table);
        });
        return;
    }
    // digits of equal width, as few as SORT_MAX_BITS allows; the key `rows` stands for absent ids
    int key_bits = 1;
    while (((int64_t)1 << key_bits) <= rows) ++key_bits;
    const int passes = (key_bits + SORT_MAX_BITS - 1) / SORT_MAX_BITS, bits = (key_bits + passes - 1) / passes;
    int64_t tile = (n + SORT_TILES - 1) / SORT_TILES;
    tile = (tile + SORT_STEP - 1) / SORT_STEP * SORT_STEP;
    const int tiles = (int)((n + tile - 1) / tile);
    auto* counts = (uint32_t*)scratch_bytes("embed_counts", ((int64_t)SORT_TILES << bits) * 4);
    auto* sorted = (uint32_t*)scratch_bytes("embed_sorted", n * 16);  // key, pos and their other halves
    uint32_t *key[2] = {sorted, sorted + 2 * n}, *pos[2] = {sorted + n, sorted + 3 * n};
    const int64_t groups = n / GROUP, groups2 = groups / GROUP;
    float* first = scratch_f32("embed_partial", std::max<int64_t>(1, (groups + groups2) * dim));
    float* second = first + groups * dim;
    for (int p = 0; p < passes; ++p) {
        const int in = (p + 1) & 1, out = p & 1, shift = p * bits;
        if (p == 0) {
            RVX_LAUNCH("embedding_sort", sort_count_kernel<true>, dim3(tiles), dim3(SORT_THREADS), 0, ids,
                       (const uint32_t*)nullptr, n, (uint32_t)rows, tile, bits, shift, counts);
            RVX_LAUNCH("embedding_sort", sort_move_kernel<true>, dim3(tiles), dim3(SORT_THREADS), 0, ids,
                       (const uint32_t*)nullptr, (const uint32_t*)nullptr, n, (uint32_t)rows, tile, tiles, bits, shift,
                       (const uint32_t*)counts, key[out], pos[out]);
        } else {
            RVX_LAUNCH("embedding_sort", sort_count_kernel<false>, dim3(tiles), dim3(SORT_THREADS), 0,
                       (const int64_t*)nullptr, (const uint32_t*)key[in], n, (uint32_t)rows, tile, bits, shift, counts);
            RVX_LAUNCH("embedding_sort", sort_move_kernel<false>, dim3(tiles), dim3(SORT_THREADS), 0,
                       (const int64_t*)nullptr, (const uint32_t*)key[in], (const uint32_t*)pos[in], n, (uint32_t)rows, tile,
                       tiles, bits, shift, (const uint32_t*)counts, key[out], pos[out]);
        }
    }
    const uint32_t *sk = key[(passes + 1) & 1], *sp = pos[(passes + 1) & 1];
    if (!accumulate) {
        const int64_t words = (rows + 31) / 32;
        auto* present = (uint32_t*)scratch_bytes("embed_present", words * 4);
        RVX_LAUNCH("embedding_zero", clear_bits_kernel,
                   dim3((unsigned)std::min<int64_t>((words + 255) / 256, 4LL * device().num_cus)), dim3(256), 0, present, words);
        RVX_LAUNCH("embedding_zero", mark_rows_kernel,
                   dim3((unsigned)std::min<int64_t>((n + 255) / 256, 4LL * device().num_cus)), dim3(256), 0, sk, n,
                   (uint32_t)rows, present);
        zero_rows(present);
    }
    typed([&](auto t, auto s, auto add) {
        using T = decltype(t);
        using S = decltype(s);
        const int slabs = (dim + Slab<T>::COLS - 1) / Slab<T>::COLS;
        auto blocks = [&](int64_t items) { return dim3((unsigned)((items + 3) / 4), slabs); };
        if (groups)
            RVX_LAUNCH("embedding_partial", (embed_partial_kernel<T, false>), blocks(groups), dim3(256), 0,
                       (const T*)grad_out, (const float*)nullptr, dim, sk, sp, groups, (uint32_t)rows, first);
        if (groups2)
            RVX_LAUNCH("embedding_partial", (embed_partial_kernel<T, true>), blocks(groups2), dim3(256), 0,
                       (const T*)grad_out, (const float*)first, dim, sk, sp, groups2, (uint32_t)rows, second);
        constexpr int64_t SLICE = (int64_t)1 << 24;  // entries of one launch: at most 2^30 threads
        for (int64_t i = 0; i < n; i += SLICE)
        RVX_LAUNCH("embedding_backward", (embed_rows_kernel<T, S, decltype(add)::value>), blocks(std::min(SLICE, n - i)),
                   dim3(256), 0, (const T*)grad_out, dim, i, sk, sp, n, (uint32_t)rows, (const float*)first,
                   (const float*)second, scale, (S*)grad_table);
    });
}

}  // namespace rvx
