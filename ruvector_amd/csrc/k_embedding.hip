// k_embedding.hip — rows of a learned table by id, and the gradient of the table.
//
// Forward: out[i] = scale * table[id_i]; one read and one write of each row, bound by HBM.
// Backward: g[v] = scale * sum_{i: id_i = v} dy[i]. The positions are grouped by id with a stable
// radix sort of (id, i) and summed in an order that depends on the ids alone: no floating-point
// atomics, the same bits every call. Sums in 32 bits, rounded once to the table's type. It cannot do
// without reading dy and writing the rows; the sort (key and position, 8 bytes, a pass) and its
// launches are what comes on top.
#include "heads.hpp"

namespace rvx {
namespace {

// N values of S as one vector (kept packed: arrays of 16-bit values are spread over registers)
template <class S, int N>
struct Pack {
    typedef S V __attribute__((ext_vector_type(N)));
};
template <class S, int N>
using PackOf = typename Pack<S, N>::V;

// Columns past dim hold anything. No lane branches, so that the loads of many rows go out together: a
// lane past the last whole vector reads the last N columns and shifts its own into place.
template <class S, int N>
__device__ __forceinline__ PackOf<S, N> get_vec(const S* row, int c, int dim) {
    PackOf<S, N> v;
    if (dim < N) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i < dim ? row[i] : (S)0.0f;  // (one vector: c is 0 or past dim)
        return v;
    }
    const int from = min(c, dim - N), shift = c - from;
    __builtin_memcpy(&v, row + from, sizeof(v));
    if (dim % N) {
#pragma unroll
        for (int st = N / 2; st > 0; st >>= 1)
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i + st < N) v[i] = shift & st ? v[i + st] : v[i];
    }
    return v;
}

// ---------------------------------------------------------------- forward
// A lane: EF_U 16-byte chunks of the output as one array, 256 chunks apart, so that short rows fill
// waves too and all loads go out before the first is used. bf16 1000000 x 768, 131072 ids: 78 to 81 us, 5
// TB/s read and written (a large copy: 4.7); 64 f32 rows of 128: 4.3 us, a launch.
constexpr int EF_U = 4;

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
    PackOf<T, N> v[EF_U];
#pragma unroll
    for (int u = 0; u < EF_U; ++u) {
        const bool there = id[u] >= 0 && id[u] < rows;
        v[u] = get_vec<T, N>(table + (there ? id[u] : 0) * dim, col[u], dim);
        if (!there) v[u] = (T)0.0f;
    }
#pragma unroll
    for (int u = 0; u < EF_U; ++u) {
        if (row[u] >= n) continue;
        PackOf<T, N> r;
#pragma unroll
        for (int j = 0; j < N; ++j) r[j] = (T)((float)v[u][j] * scale);
        T* o = out + row[u] * dim + col[u];
        if (col[u] + N <= (uint32_t)dim) __builtin_memcpy(o, &r, 16);
        else
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (col[u] + j < (uint32_t)dim) o[j] = r[j];
    }
}

// ---------------------------------------------------------------- grouping positions by id
// Stable LSD radix sort of (key, position), key = id, or `rows` for an absent id. The n positions
// are cut into at most SORT_TILES tiles, one block each. A pass is two launches: every tile counts
// its digits in LDS, then moves its elements; for that each block sums the counts of the tiles
// before it by itself, which costs less than a launch for a scan. Bound by the latency of 64 blocks'
// steps: 100003 positions of 500009 rows, two passes of 10 bits, 31 us. (Counting by atomics in memory: 587 us
// for the bf16 gradient below that took 311 with the counts in LDS, ids as frequent as words.) Digits
// of at most 11 bits: 8 waves' counters of 2^11 fit LDS.
constexpr int SORT_TILES = 64, SORT_THREADS = 512, SORT_WAVES = SORT_THREADS / 64, SORT_STEP = SORT_THREADS * 4;
constexpr int SORT_MAX_BITS = 11, SORT_BINS = 1 << SORT_MAX_BITS;

__device__ __forceinline__ uint32_t sort_key(const int64_t* ids, int64_t i, uint32_t rows) {
    const int64_t id = ids[i];
    return id >= 0 && id < (int64_t)rows ? (uint32_t)id : rows;
}

// the block-th of `blocks` blocks' share of setting bytes (an even number of them) to 0
__device__ __forceinline__ void zero_bytes(unsigned char* p, int64_t bytes, int block, int blocks) {
    const int64_t step = (int64_t)blocks * blockDim.x * 16;
    const uint4 z = {0, 0, 0, 0};
    int64_t b = ((int64_t)block * blockDim.x + threadIdx.x) * 16;
    for (; b + 3 * step + 16 <= bytes; b += 4 * step)
#pragma unroll
        for (int u = 0; u < 4; ++u) __builtin_memcpy(p + b + u * step, &z, 16);
    for (; b + 16 <= bytes; b += step) __builtin_memcpy(p + b, &z, 16);
    if (b < bytes)
        for (; b < bytes; b += 2) *(uint16_t*)(p + b) = 0;
}

// counts[tile][digit]; clear: nullable, words to set to 0
template <bool FIRST>
__global__ __launch_bounds__(SORT_THREADS) void sort_count_kernel(const int64_t* __restrict__ ids,
                                                                 const uint32_t* __restrict__ key_in, int64_t n,
                                                                 uint32_t rows, int64_t tile, int bits, int shift,
                                                                 uint32_t* __restrict__ counts, uint32_t* clear,
                                                                 int64_t words) {
    for (int64_t i = (int64_t)blockIdx.x * SORT_THREADS + threadIdx.x; clear && i < words; i += gridDim.x * SORT_THREADS)
        clear[i] = 0;
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
    __shared__ uint32_t sums[SORT_WAVES];
    const int bins = 1 << bits, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int me = blockIdx.x;
    // base[d] = elements of smaller digits anywhere + of digit d in the tiles before
    constexpr int PER = SORT_BINS / SORT_THREADS;
    uint32_t total[PER] = {}, ahead[PER] = {}, sum = 0;
    if (t * PER < bins) {  // bins are a multiple of PER
        const uint32_t* c = counts + t * PER;
#pragma unroll 8
        for (int b = 0; b < tiles; ++b) {
            uint32_t v[PER];
            __builtin_memcpy(v, c + ((int64_t)b << bits), sizeof(v));
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                total[j] += v[j];
                ahead[j] += b < me ? v[j] : 0;
            }
        }
#pragma unroll
        for (int j = 0; j < PER; ++j) sum += total[j];
    }
    uint32_t scan = sum;  // over the wave's lanes, then over the waves
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t v = __shfl_up(scan, o);
        scan += lane >= o ? v : 0;
    }
    if (lane == 63) sums[wave] = scan;
    __syncthreads();
    uint32_t run = scan - sum;
    for (int w = 0; w < wave; ++w) run += sums[w];
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
            wave_lds_order();
            if (there && before == 0) mine[wave][d] = to + __popcll(same);
            wave_lds_order();
            if (there) {
                key_out[to] = key[u];
                pos_out[to] = pos[u];
            }
        }
    }
}

// Up to SMALL_SORT positions: one block sorts them in LDS, in one launch; the other blocks meanwhile
// set `clear` (nullable) to zeros. Against the passes over tiles, whole gradient f32 of 100000 x 128: 17
// us to 23 at 2000 positions, 25.4 to 26.6 at 6144, 32 to 30 at 8192.
constexpr int SMALL_SORT = 6144, SMALL_BITS = 9, SMALL_THREADS = 1024, SMALL_WAVES = SMALL_THREADS / 64;

__global__ __launch_bounds__(SMALL_THREADS) void sort_small_kernel(const int64_t* __restrict__ ids, int n, uint32_t rows,
                                                                  int passes, int bits, uint32_t* __restrict__ key_out,
                                                                  uint32_t* __restrict__ pos_out, unsigned char* clear,
                                                                  int64_t clear_bytes) {
    __shared__ uint32_t key[2][SMALL_SORT];
    __shared__ uint16_t pos[2][SMALL_SORT];
    __shared__ uint32_t mine[SMALL_WAVES][1 << SMALL_BITS];
    __shared__ uint32_t sums[(1 << SMALL_BITS) / 64];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    if (blockIdx.x > 0) {
        zero_bytes(clear, clear_bytes, blockIdx.x - 1, gridDim.x - 1);
        return;
    }
    for (int i = t; i < n; i += SMALL_THREADS) {
        key[0][i] = sort_key(ids, i, rows);
        pos[0][i] = (uint16_t)i;
    }
    const int bins = 1 << bits, chunk = (n + SMALL_THREADS - 1) / SMALL_THREADS * 64;  // a wave's elements, in order
    const int lo = wave * chunk, hi = min(n, lo + chunk);
    for (int p = 0; p < passes; ++p) {
        const int in = p & 1, shift = p * bits;
        for (int i = t; i < SMALL_WAVES << bits; i += SMALL_THREADS) mine[i >> bits][i & (bins - 1)] = 0;
        __syncthreads();
        for (int i = lo + lane; i < hi; i += 64) atomicAdd(&mine[wave][(key[in][i] >> shift) & (bins - 1)], 1u);
        __syncthreads();
        // a digit's places: those of smaller digits, then of this one wave by wave
        uint32_t count[SMALL_WAVES], total = 0;
        if (t < bins)
#pragma unroll
            for (int w = 0; w < SMALL_WAVES; ++w) count[w] = mine[w][t];
        if (t < bins)
#pragma unroll
            for (int w = 0; w < SMALL_WAVES; ++w) total += count[w];
        uint32_t scan = total;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t v = __shfl_up(scan, o);
            scan += lane >= o ? v : 0;
        }
        if (lane == 63 && wave < (1 << SMALL_BITS) / 64) sums[wave] = scan;
        __syncthreads();
        if (t < bins) {
            uint32_t from = scan - total;
            for (int w = 0; w < wave; ++w) from += sums[w];
#pragma unroll
            for (int w = 0; w < SMALL_WAVES; ++w) {
                mine[w][t] = from;
                from += count[w];
            }
        }
        __syncthreads();
        for (int i0 = lo; i0 < hi; i0 += 64) {
            const int i = i0 + lane;
            const bool there = i < hi;
            const uint32_t k = there ? key[in][i] : 0, d = (k >> shift) & (bins - 1);
            unsigned long long same = __ballot(there);
            for (int b = 0; b < bits; ++b) {
                const unsigned long long m = __ballot((d >> b) & 1);
                same &= (d >> b) & 1 ? m : ~m;
            }
            const int before = __popcll(same & ((1ull << lane) - 1));
            uint32_t to = 0;
            if (there) to = mine[wave][d] + before;
            wave_lds_order();
            if (there && before == 0) mine[wave][d] = to + __popcll(same);
            wave_lds_order();
            if (there) {
                if (p + 1 < passes) {
                    key[1 - in][to] = k;
                    pos[1 - in][to] = pos[in][i];
                } else {
                    key_out[to] = k;
                    pos_out[to] = pos[in][i];
                }
            }
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- sums over groups
// An id's entries are a run of the sorted order. A run of fewer than LONG entries is summed by one
// wave per slab of columns, in order. A longer one is cut where the order is, into groups of GROUP
// entries: a group's part of its first key's run (`tails`) and of its last key's (`heads`, where
// that is another key) are summed by a wave of their own, GROUP whole tails of one run once more
// (`spans`), and the wave of the run's first group adds these. (A run of LONG entries touches an end
// of its group.) Groups and order depend on the sorted ids alone. Ids as frequent as words, bf16 65536
// x 1024: the rows kernel alone, one wave for the most frequent id, took 311 us of a gradient that takes 183
// (167 with uniform ids).
constexpr int GROUP = 64, LONG = 63;

// A wave's columns of a row: V vectors of N columns a lane, vector q at (q * 64 + lane) * N.
template <class S, int N, int V>
__device__ __forceinline__ void get_cols(const S* row, PackOf<S, N> (&v)[V], int col, int dim) {
#pragma unroll
    for (int q = 0; q < V; ++q) v[q] = get_vec<S, N>(row, col + q * 64 * N, dim);
}
template <class S, int N, int V>
__device__ __forceinline__ void put_cols(S* row, const PackOf<S, N> (&v)[V], int col, int dim) {
#pragma unroll
    for (int q = 0; q < V; ++q) {
        const int c = col + q * 64 * N;
        if (c + N <= dim) __builtin_memcpy(row + c, &v[q], sizeof(S) * N);
        else
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (c + i < dim) row[c + i] = v[q][i];
    }
}
// acc += the wave's columns of rows [j, count), row_of(j) in turn (the same in all lanes): U rows in
// flight while there are U, then U / 2 ..
template <int U, class S, int N, int V, class F>
__device__ __forceinline__ void add_rows(PackOf<float, N> (&acc)[V], int count, int col, int dim, F&& row_of, int j = 0) {
    for (; j + U <= count; j += U) {
        PackOf<S, N> v[U][V];
#pragma unroll
        for (int u = 0; u < U; ++u) get_cols<S, N, V>(row_of(j + u), v[u], col, dim);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int q = 0; q < V; ++q)
#pragma unroll
                for (int i = 0; i < N; ++i) acc[q][i] += (float)v[u][q][i];
    }
    if constexpr (U > 1) add_rows<U / 2, S, N, V>(acc, count, col, dim, row_of, j);
}
// how many lanes from lane 0 on hold `on`
__device__ __forceinline__ int leading(bool on) {
    const int first = __ffsll(~__ballot(on)) - 1;
    return first < 0 ? 64 : first;
}

// What a wave sees of group g and of the groups beside it.
struct Group {
    uint32_t first, last;      // its first and last key
    int lead, trail;           // entries of either in it; trail counts the last key only where it is another
    int came, goes;            // entries of the first key just before it, of the last just after it, up to 64
    uint32_t key, pos;         // this lane's entry
    __device__ __forceinline__ Group(const uint32_t* __restrict__ keys, const uint32_t* __restrict__ poss, int64_t n,
                                     int64_t g) {
        const int lane = threadIdx.x & 63;
        const int64_t i = g * GROUP + lane;
        const uint32_t none = 0xffffffffu;  // no key is that large
        key = i < n ? keys[i] : none;
        pos = i < n ? poss[i] : 0;
        const uint32_t before = i >= GROUP ? keys[i - GROUP] : none;
        const uint32_t after = i + GROUP < n ? keys[i + GROUP] : none;
        first = __builtin_amdgcn_readlane(key, 0), last = __builtin_amdgcn_readlane(key, 63);
        lead = leading(key == first);
        trail = lead == 64 ? 0 : __clzll(~__ballot(key == last));
        const unsigned long long back = ~__ballot(before == first);
        came = back ? __clzll(back) : 64;
        goes = leading(after == last);
    }
    __device__ __forceinline__ bool long_first(uint32_t rows) const {
        return first < rows && came + lead + (lead == 64 ? goes : 0) >= LONG;
    }
    __device__ __forceinline__ bool long_last(uint32_t rows) const { return last < rows && trail > 0 && trail + goes >= LONG; }
};

// One wave per (group, slab): the group's parts of long runs. present (nullable): a 1 for every row that is
// looked up, from the first entry of its run.
template <class T>
__global__ __launch_bounds__(64) void embed_groups_kernel(const T* __restrict__ grad_out, int dim,
                                                         const uint32_t* __restrict__ key,
                                                         const uint32_t* __restrict__ pos, int64_t n, uint32_t rows,
                                                         float* __restrict__ heads, float* __restrict__ tails,
                                                         unsigned char* __restrict__ present) {
    constexpr int N = Vec16<T>::N;
    const int64_t g = blockIdx.x;
    const int lane = threadIdx.x;
    const Group at(key, pos, n, g);
    if (present && blockIdx.y == 0) {
        const uint32_t left = __shfl_up(at.key, 1);
        if (at.key < rows && (lane ? left != at.key : at.came == 0)) present[at.key] = 1;
    }
    const int col = blockIdx.y * 64 * N + lane * N;
    auto sum = [&](int from, int count, float* out) {
        PackOf<float, N> acc[1] = {};
        add_rows<32, T, N, 1>(acc, count, col, dim, [&](int j) {
            return grad_out + (int64_t)(uint32_t)__builtin_amdgcn_readlane(at.pos, from + j) * dim;
        });
        put_cols<float, N, 1>(out + g * dim, acc, col, dim);
    };
    if (at.long_first(rows)) sum(0, at.lead, tails);
    if (at.long_last(rows)) sum(64 - at.trail, at.trail, heads);
}

// One wave per (GROUP groups, slab) that one run fills and began before: the sum of their tails.
__global__ __launch_bounds__(256) void embed_spans_kernel(const float* __restrict__ tails, int dim,
                                                         const uint32_t* __restrict__ key, int64_t spans, uint32_t rows,
                                                         float* __restrict__ out) {
    const int lane = threadIdx.x & 63;
    const int64_t s = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (s >= spans || s == 0) return;
    const int64_t at = s * GROUP * GROUP;
    const uint32_t k = key[at];
    if (k >= rows || key[at - 1] != k || key[at + GROUP * GROUP - 1] != k) return;
    const int col = blockIdx.y * 64 * 4 + lane * 4;
    PackOf<float, 4> acc[1] = {};
    add_rows<8, float, 4, 1>(acc, GROUP, col, dim, [&](int j) { return tails + (s * GROUP + j) * dim; });
    put_cols<float, 4, 1>(out + s * dim, acc, col, dim);
}

// row = scale * acc (+ row)
template <class S, int N, int V>
__device__ __forceinline__ void finish_row(S* row, const PackOf<float, N> (&acc)[V], const PackOf<S, N> (&old)[V], int col, int dim,
                                           float scale) {
    PackOf<S, N> v[V];
#pragma unroll
    for (int q = 0; q < V; ++q)
#pragma unroll
        for (int i = 0; i < N; ++i) v[q][i] = (S)fmaf(acc[q][i], scale, (float)old[q][i]);
    put_cols<S, N, V>(row, v, col, dim);
}

// One wave per (group, slab): the rows of the long runs that begin in the group.
template <class T, class S>
__global__ __launch_bounds__(64) void embed_long_kernel(int dim, const uint32_t* __restrict__ key,
                                                       const uint32_t* __restrict__ pos, int64_t n, uint32_t rows,
                                                       const float* __restrict__ heads, const float* __restrict__ tails,
                                                       const float* __restrict__ spans, float scale, bool add,
                                                       S* grad_table) {
    constexpr int N = Vec16<T>::N;
    const int lane = threadIdx.x;
    const Group here(key, pos, n, blockIdx.x);
    const int col = blockIdx.y * 64 * N + lane * N;
    const int64_t whole_spans = n / (GROUP * GROUP);
    auto run = [&](uint32_t k, const float* part, bool on) {  // on: the run leaves the group
        S* const row = grad_table + (int64_t)k * dim;
        PackOf<S, N> old[1] = {};
        if (add) get_cols<S, N, 1>(row, old, col, dim);
        PackOf<float, N> acc[1] = {};
        add_rows<1, float, N, 1>(acc, 1, col, dim, [&](int) { return part + (int64_t)blockIdx.x * dim; });
        for (int64_t g = blockIdx.x + 1; on && g * GROUP < n;) {
            if ((g & (GROUP - 1)) == 0 && g / GROUP < whole_spans) {
                const int64_t s = g / GROUP;
                const int count = leading(s + lane < whole_spans && key[(s + lane + 1) * GROUP * GROUP - 1] == k);
                if (count) {
                    add_rows<8, float, N, 1>(acc, count, col, dim, [&](int j) { return spans + (s + j) * dim; });
                    g += (int64_t)count * GROUP;
                    continue;
                }
            }
            // tails up to the next span's begin: a group has one if its first entry is the id's
            const int most = GROUP - (int)(g & (GROUP - 1));
            const int count = leading(lane < most && (g + lane) * GROUP < n && key[(g + lane) * GROUP] == k);
            add_rows<8, float, N, 1>(acc, count, col, dim, [&](int j) { return tails + (g + j) * dim; });
            g += count;
            on = count == most;
        }
        finish_row<S, N, 1>(row, acc, old, col, dim, scale);
    };
    if (here.came == 0 && here.long_first(rows)) run(here.first, tails, here.lead == 64 && here.goes > 0);
    if (here.long_last(rows)) run(here.last, heads, here.goes > 0);
}

// The block-th of `blocks` blocks' share of the rows that are not marked: zeros.
__device__ __forceinline__ void zero_rows(unsigned char* table, int64_t rows, int64_t row_bytes,
                                          const unsigned char* __restrict__ present, int block, int blocks) {
    const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
    const int64_t step = (int64_t)blocks * waves;
    const uint4 z = {0, 0, 0, 0};
    for (int64_t w = (int64_t)block * waves + (threadIdx.x >> 6); w * 64 < rows; w += step) {  // 64 rows a turn
        unsigned long long absent = __ballot(w * 64 + lane < rows && !present[w * 64 + lane]);
        while (absent) {
            unsigned char* p = table + (w * 64 + __ffsll(absent) - 1) * row_bytes;
            absent &= absent - 1;
            int64_t b = (int64_t)lane * 16;
            for (; b + 16 <= row_bytes; b += 64 * 16) __builtin_memcpy(p + b, &z, 16);
            if (b < row_bytes)
                for (; b < row_bytes; b += 2) *(uint16_t*)(p + b) = 0;
        }
    }
}

// One wave per (sorted entry, slab): the first entry of an id sums the id's run into its row. Bound
// by HBM: a wave takes up to 4 vectors a lane, so that a row's bytes are all in flight at once; f32
// 500009 x 768, 100003 ids, added to the table: 4.9 TB/s. The first zero_blocks blocks set the
// rows without an entry to zeros meanwhile: bf16 262144 x 1024, 65536 uniform ids: 167 us, 181 with these in a
// launch on a second stream; bf16 512 columns, 20000 ids, a table of 512 MB: 129 us, 148 and, with the whole
// table cleared before, 154; of 64 MB: 41, 63 and 49.
template <class T, class S, int V>
__global__ __launch_bounds__(256) void embed_rows_kernel(const T* __restrict__ grad_out, int dim, int64_t begin,
                                                        const uint32_t* __restrict__ key,
                                                        const uint32_t* __restrict__ pos, int64_t n, uint32_t rows,
                                                        float scale, bool add, S* grad_table, int zero_blocks,
                                                        const unsigned char* __restrict__ present) {
    constexpr int N = Vec16<T>::N;
    const int lane = threadIdx.x & 63;
    if ((int)blockIdx.x < zero_blocks) {
        if (blockIdx.y == 0)
            zero_rows((unsigned char*)grad_table, rows, (int64_t)dim * (int64_t)sizeof(S), present, blockIdx.x, zero_blocks);
        return;
    }
    const int64_t i0 = begin + (int64_t)(blockIdx.x - zero_blocks) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (i0 >= n) return;
    // one load gives the entry before, this one and the 62 after it
    const int64_t near_i = i0 + lane - 1;
    const uint32_t near_key = near_i >= 0 && near_i < n ? key[near_i] : 0xffffffffu;  // no key is that large
    const uint32_t near_pos = near_i >= 0 && near_i < n ? pos[near_i] : 0;
    const uint32_t k = __builtin_amdgcn_readlane(near_key, 1);
    if (k >= rows || (uint32_t)__builtin_amdgcn_readlane(near_key, 0) == k) return;
    const unsigned long long others = __ballot(lane > 0 && near_key != k);
    if (!others) return;  // LONG entries or more
    const int run = __ffsll(others) - 2;
    const int col = blockIdx.y * 64 * N * V + lane * N;
    S* const row = grad_table + (int64_t)k * dim;
    PackOf<S, N> old[V] = {};
    if (add) get_cols<S, N, V>(row, old, col, dim);  // does not wait for the sum
    PackOf<float, N> acc[V] = {};
    add_rows<(V == 1 ? 8 : V == 2 ? 4 : 2), T, N, V>(acc, run, col, dim, [&](int j) {
        return grad_out + (int64_t)(uint32_t)__builtin_amdgcn_readlane(near_pos, j + 1) * dim;
    });
    finish_row<S, N, V>(row, acc, old, col, dim, scale);
}

// Few positions: no sort. The block of position i and a slab of columns looks for its id among all
// positions, 64 a wave and turn: before i (then another block has the row), and from i on, whose rows
// each wave adds in order; the waves' sums are added in theirs. Against the sort: bf16 of 1024 columns,
// 1000 positions: 7.7 us to 13.6 (20000 ids), 6.3 to 15.6 (40 ids), 28 to 18 (one id); 2000: 16.3 to
// 15.4. Eight waves a block: 11.3, 6.1 and 20.7 us at 1000; one: 6.4, 11.7 and 137.
constexpr int SCAN_MAX = 1024, SCAN_WAVES = 4;

template <class T, class S>
__global__ __launch_bounds__(64 * SCAN_WAVES) void embed_scan_kernel(const T* __restrict__ grad_out, int dim,
                                                                    const int64_t* __restrict__ ids, int n, int64_t rows,
                                                                    float scale, bool add, S* grad_table) {
    constexpr int N = Vec16<T>::N;
    __shared__ float sums[SCAN_WAVES][64 * N];
    __shared__ int counts[SCAN_WAVES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i0 = blockIdx.x;
    const int64_t id = ids[i0];
    if (id < 0 || id >= rows) return;
    bool before = false;
    for (int p = wave * 64 + lane; p < i0; p += 64 * SCAN_WAVES) before |= ids[p] == id;
    if (__syncthreads_or(before)) return;
    // a thread's columns of the sums (of the rows': lane * N ..)
    constexpr int THREADS = 64 * SCAN_WAVES, OWN = (64 * N + THREADS - 1) / THREADS;
    const int col0 = blockIdx.y * 64 * N;
    S* const row = grad_table + id * dim + col0;
    auto mine = [&](int q) { return (int)threadIdx.x + q * THREADS; };
    auto there = [&](int q) { return mine(q) < 64 * N && col0 + mine(q) < dim; };
    float old[OWN];  // does not wait for the sum
#pragma unroll
    for (int q = 0; q < OWN; ++q) old[q] = add && there(q) ? (float)row[mine(q)] : 0.0f;
    PackOf<float, N> acc[1] = {};
    int found = 0;
    for (int j = wave * 64; j < n; j += 64 * SCAN_WAVES) {
        const int p = j + lane;
        const unsigned long long m = __ballot(p >= i0 && p < n && ids[p] == id);
        const int count = __popcll(m);
        if (!count) continue;
        // lane r: the r-th of these positions
        const int below = __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
        const int place = __builtin_amdgcn_ds_permute((m >> lane & 1 ? below : count + lane - below) * 4, p);
        add_rows<16, T, N, 1>(acc, count, col0 + lane * N, dim,
                              [&](int r) { return grad_out + (int64_t)__builtin_amdgcn_readlane(place, r) * dim; });
        found += count;
    }
    if (found) __builtin_memcpy(&sums[wave][lane * N], &acc[0], sizeof(acc[0]));
    if (lane == 0) counts[wave] = found;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < OWN; ++q) {
        if (!there(q)) continue;
        float sum = 0.0f;
        for (int w = 0; w < SCAN_WAVES; ++w)
            if (counts[w]) sum += sums[w][mine(q)];
        row[mine(q)] = (S)fmaf(sum, scale, old[q]);
    }
}

// The whole table: zeros.
__global__ __launch_bounds__(256) void embed_zero_kernel(unsigned char* table, int64_t bytes) {
    zero_bytes(table, bytes, blockIdx.x, gridDim.x);
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
    const int64_t table_bytes = rows * dim * dtype_size(table_dtype);
    auto zero_table = [&] {
        const int64_t blocks = std::min<int64_t>((table_bytes + 4095) / 4096, 8LL * device().num_cus);
        RVX_LAUNCH("embedding_zero", embed_zero_kernel, dim3((unsigned)blocks), dim3(256), 0, (unsigned char*)grad_table,
                   table_bytes);
    };
    auto typed = [&](auto&& f) {  // f(T, S) of the gradient's and the table's type
        with_dtype(dtype, [&](auto t) { with_dtype(table_dtype, [&](auto s) { f(t, s); }); });
    };
    if (n <= SCAN_MAX) {
        if (!accumulate) zero_table();
        if (n == 0) return;
        typed([&](auto t, auto s) {
            using T = decltype(t);
            using S = decltype(s);
            const int slabs = (dim + 64 * Vec16<T>::N - 1) / (64 * Vec16<T>::N);
            RVX_LAUNCH("embedding_backward", (embed_scan_kernel<T, S>),
                       dim3((unsigned)n, slabs), dim3(64 * SCAN_WAVES), 0, (const T*)grad_out, dim, ids, (int)n,
                       rows, scale, accumulate, (S*)grad_table);
        });
        return;
    }
    // digits of equal width, as few as SORT_MAX_BITS allows; the key `rows` stands for absent ids
    int key_bits = 1;
    while (((int64_t)1 << key_bits) <= rows) ++key_bits;
    auto* sorted = (uint32_t*)scratch_bytes("embed_sorted", n * 16);  // key, pos and their other halves
    uint32_t *key[2] = {sorted, sorted + 2 * n}, *pos[2] = {sorted + n, sorted + 3 * n};
    const uint32_t *sk, *sp;
    const int64_t groups = (n + GROUP - 1) / GROUP, span_count = n / (GROUP * GROUP);
    float* heads = scratch_f32("embed_partial", (2 * groups + span_count) * dim);
    float *tails = heads + groups * dim, *spans = tails + groups * dim;
    // A dense gradient's other rows become zeros beside other work: of few positions the whole table
    // beside the sort, by blocks that it leaves idle; of many, the rows without an id beside the sums.
    const bool beside = !accumulate && n > SMALL_SORT;
    const int64_t words = (rows + 3) / 4;
    auto* present = beside ? (uint32_t*)scratch_bytes("embed_present", words * 4) : nullptr;  // a byte a row
    if (n <= SMALL_SORT) {
        const int passes = (key_bits + SMALL_BITS - 1) / SMALL_BITS, bits = (key_bits + passes - 1) / passes;
        unsigned char* clear = accumulate ? nullptr : (unsigned char*)grad_table;
        const int64_t bytes = accumulate ? 0 : table_bytes;
        const int64_t blocks = std::min<int64_t>((bytes + 16383) / 16384, 2LL * device().num_cus);
        RVX_LAUNCH("embedding_sort", sort_small_kernel, dim3((unsigned)(1 + blocks)), dim3(SMALL_THREADS), 0, ids, (int)n,
                   (uint32_t)rows, passes, bits, key[0], pos[0], clear, bytes);
        sk = key[0], sp = pos[0];
    } else {
        const int passes = (key_bits + SORT_MAX_BITS - 1) / SORT_MAX_BITS;
        const int bits = std::max(2, (key_bits + passes - 1) / passes);  // at least the 4 digits of a thread
        int64_t tile = (n + SORT_TILES - 1) / SORT_TILES;
        tile = (tile + SORT_STEP - 1) / SORT_STEP * SORT_STEP;
        const int tiles = (int)((n + tile - 1) / tile);
        auto* counts = (uint32_t*)scratch_bytes("embed_counts", ((int64_t)SORT_TILES << bits) * 4);
        for (int p = 0; p < passes; ++p) {
            const int in = (p + 1) & 1, out = p & 1, shift = p * bits;
            if (p == 0) {
                RVX_LAUNCH("embedding_count", sort_count_kernel<true>, dim3(tiles), dim3(SORT_THREADS), 0, ids,
                           (const uint32_t*)nullptr, n, (uint32_t)rows, tile, bits, shift, counts, present, words);
                RVX_LAUNCH("embedding_sort", sort_move_kernel<true>, dim3(tiles), dim3(SORT_THREADS), 0, ids,
                           (const uint32_t*)nullptr, (const uint32_t*)nullptr, n, (uint32_t)rows, tile, tiles, bits, shift,
                           (const uint32_t*)counts, key[out], pos[out]);
            } else {
                RVX_LAUNCH("embedding_count", sort_count_kernel<false>, dim3(tiles), dim3(SORT_THREADS), 0,
                           (const int64_t*)nullptr, (const uint32_t*)key[in], n, (uint32_t)rows, tile, bits, shift, counts,
                           nullptr, (int64_t)0);
                RVX_LAUNCH("embedding_sort", sort_move_kernel<false>, dim3(tiles), dim3(SORT_THREADS), 0,
                           (const int64_t*)nullptr, (const uint32_t*)key[in], (const uint32_t*)pos[in], n, (uint32_t)rows,
                           tile, tiles, bits, shift, (const uint32_t*)counts, key[out], pos[out]);
            }
        }
        sk = key[(passes + 1) & 1], sp = pos[(passes + 1) & 1];
    }
    const int zero_blocks = beside ? (int)std::min<int64_t>((rows + 255) / 256, (int64_t)device().num_cus) : 0;
    typed([&](auto t, auto s) {
        using T = decltype(t);
        using S = decltype(s);
        constexpr int N = Vec16<T>::N;
        const int vecs = (dim + 64 * N - 1) / (64 * N);  // vectors a lane for a whole row
        RVX_LAUNCH("embedding_groups", embed_groups_kernel<T>, dim3((unsigned)groups, vecs), dim3(64), 0, (const T*)grad_out,
                   dim, sk, sp, n, (uint32_t)rows, heads, tails, (unsigned char*)present);
        if (span_count > 1)
            RVX_LAUNCH("embedding_long", embed_spans_kernel, dim3((unsigned)((span_count + 3) / 4), (dim + 255) / 256),
                       dim3(256), 0, (const float*)tails, dim, sk, span_count, (uint32_t)rows, spans);
        RVX_LAUNCH("embedding_long", (embed_long_kernel<T, S>), dim3((unsigned)groups, vecs), dim3(64), 0, dim, sk, sp, n,
                   (uint32_t)rows, (const float*)heads, (const float*)tails, (const float*)spans, scale, accumulate,
                   (S*)grad_table);
        const int slabs = (vecs + 3) / 4, per = (vecs + slabs - 1) / slabs;
        auto go = [&](auto v) {
            constexpr int64_t SLICE = (int64_t)1 << 24;  // entries of one launch: at most 2^30 threads
            for (int64_t i = 0; i < n; i += SLICE) {
                const int zeros = i ? 0 : zero_blocks;
                RVX_LAUNCH("embedding_backward", (embed_rows_kernel<T, S, decltype(v)::value>),
                           dim3((unsigned)((std::min(SLICE, n - i) + 3) / 4 + zeros), slabs), dim3(256), 0, (const T*)grad_out,
                           dim, i, sk, sp, n, (uint32_t)rows, scale, accumulate, (S*)grad_table, zeros,
                           (const unsigned char*)present);
            }
        };
        if (per == 1) go(std::integral_constant<int, 1>{});
        else if (per == 2) go(std::integral_constant<int, 2>{});
        else if (per == 3) go(std::integral_constant<int, 3>{});
        else go(std::integral_constant<int, 4>{});
    });
}

}  // namespace rvx
