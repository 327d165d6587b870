// k_adapter.hip — y_i = W x_i + bias + s_r B_r (A_r x_i) with r = ids[i], the adapter of row i.
//
// t_i = s_r A_r x_i for every row is a launch of its own; the projection adds B_r t_i behind its
// sum. Rows may come in any order of adapters. For more than a few rows they are first grouped: the
// kernels then go through a permutation of the rows, in which a 16-row tile holds one adapter or
// two, and take one turn for each. The products of a row do not depend on its place.
//
// All operands lie in fragment order: the 16 rows x 64 bytes that one matrix instruction takes from
// one operand are 1 KiB, lane l's 16 bytes at l * 16 (row l % 16, elements (l / 16) * N ..). A
// wave loads a fragment with one coalesced instruction, copies it to LDS as it is, and reads it
// back without bank conflicts. Weights are laid out when they are set, x by the launch that computes
// t, which reads it anyway: a CU takes 75 to 110 bytes a ns from L2 in whole KiB, but only 35 where
// each load gathers 16 rows, and the projection reads x many times (bf16 4096 x 4096, 8192 rows: 299 us
// with x read as it lies, 256 so). W and B are the first operand, x and t the second, so that a lane
// holds 4 outputs of one row; the 32 outputs of two neighbouring fragments are interleaved by 4
// (`out_of`), so that the two give it 8 neighbouring outputs. Along `in`, two neighbouring fragments
// are interleaved by pieces (`in_of`): a row's two pieces of one lane are neighbours, and the loads of
// a pair touch whole 128-byte lines of x.
#include "adapter.hpp"

namespace rvx {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// One 16-byte piece of an operand and the product of two fragments, acc += A B^T: lane l holds
// C[4 (l / 16) + r][l % 16], r < 4.
template <class T>
struct Mma;
template <>
struct Mma<__bf16> {
    using V = bf16x8;
    __device__ static f32x4 run(V a, V b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Mma<_Float16> {
    using V = f16x8;
    __device__ static f32x4 run(V a, V b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Mma<float> {  // four products of depth 4: the j-th takes element j of every lane's piece
    using V = f32x4;
    __device__ static f32x4 run(V a, V b, f32x4 c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
        return c;
    }
};
template <class T>
constexpr int PIECE = 16 / (int)sizeof(T);  // elements of a lane's piece
template <class T>
constexpr int DEPTH = 4 * PIECE<T>;         // elements of a fragment along the sum

template <class T>
__device__ __forceinline__ typename Mma<T>::V load_piece(const T* p) {
    typename Mma<T>::V v;
    __builtin_memcpy(&v, p, 16);
    return v;
}

// ---------------------------------------------------------------- layout
// the output in row m of fragment tile nt
__host__ __device__ __forceinline__ int out_of(int nt, int m) {
    return (nt >> 1) * 32 + (m >> 2) * 8 + (nt & 1) * 4 + (m & 3);
}

// where piece `lane / 16` of fragment f begins along `in` (an even number of fragments)
template <class T>
__host__ __device__ __forceinline__ int in_of(int f, int piece) {
    return (f >> 1) * (2 * DEPTH<T>)+piece * (2 * PIECE<T>)+(f & 1) * PIECE<T>;
}

enum { PACK_W, PACK_A, PACK_B };  // W [out][in], A [rank][in], B [out][rank]

template <class T>
__global__ __launch_bounds__(256) void pack_kernel(const T* __restrict__ src, int rows, int cols, int64_t pieces,
                                                  int frags, int what, T* __restrict__ dst) {
    constexpr int N = PIECE<T>;
    const int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (p >= pieces) return;
    const int lane = (int)(p & 63);
    const int64_t f = p >> 6;
    const int tile = (int)(f / frags), row = what == PACK_A ? tile * 16 + (lane & 15) : out_of(tile, lane & 15);
    const int frag = (int)(f % frags), col = what == PACK_B ? frag * DEPTH<T> + (lane >> 4) * N : in_of<T>(frag, lane >> 4);
    T v[N];
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = row < rows && col + j < cols ? src[(int64_t)row * cols + col + j] : (T)0.0f;
    __builtin_memcpy(dst + p * N, v, 16);
}

__device__ __forceinline__ int adapter_of(const int32_t* ids, const AdapterSlot* slot, int slots, int64_t row, int64_t n) {
    if (!ids || row >= n) return -1;
    const int id = ids[row];
    return id >= 0 && id < slots && slot[id].rank > 0 ? id : -1;
}

// ---------------------------------------------------------------- grouping rows
// perm: GROUP_ROWS rows at a time, a block each, in the order of their adapters (adapters that agree
// modulo GROUP_BINS - 1 may mix: the order is for speed alone). f16 2048 x 2048, rank 64, 2000 rows of 32
// adapters in turn: 517 us without, 67 with it at the time.
constexpr int GROUP_THREADS = 1024, GROUP_ROWS = 2 * GROUP_THREADS, GROUP_BITS = 9, GROUP_BINS = 1 << GROUP_BITS;

__global__ __launch_bounds__(GROUP_THREADS) void group_rows_kernel(const int32_t* __restrict__ ids, int64_t n,
                                                                  int slots, int bits, int32_t* __restrict__ perm) {
    __shared__ int next[GROUP_BINS];
    __shared__ int sums[GROUP_BINS / 64];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    auto bin_of = [&](int64_t row) {
        const int id = row < n ? ids[row] : -1;
        return id < 0 || id >= slots ? 0 : 1 + id % (GROUP_BINS - 1);
    };
    // the wave's lanes with the same bin: the first of them takes places for all
    auto places = [&](int bin, bool there) {
        unsigned long long same = __ballot(there);
        for (int b = 0; b < bits; ++b) {  // bits: of the largest bin there can be
            const unsigned long long m = __ballot(bin >> b & 1);
            same &= bin >> b & 1 ? m : ~m;
        }
        const int before = __popcll(same & ((1ull << lane) - 1));
        int at = 0;
        if (there && before == 0) at = atomicAdd(&next[bin], __popcll(same));
        return __shfl(at, there ? __ffsll(same) - 1 : lane) + before;
    };
    const int64_t row0 = (int64_t)blockIdx.x * GROUP_ROWS;
    constexpr int U = GROUP_ROWS / GROUP_THREADS;
    int bin[U];
#pragma unroll
    for (int u = 0; u < U; ++u) bin[u] = bin_of(row0 + u * GROUP_THREADS + t);
    for (int b = t; b < GROUP_BINS; b += GROUP_THREADS) next[b] = 0;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u) places(bin[u], row0 + u * GROUP_THREADS + t < n);
    __syncthreads();
    int v = 0, scan = 0;
    if (t < GROUP_BINS) {
        v = scan = next[t];
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int u = __shfl_up(scan, o);
            scan += lane >= o ? u : 0;
        }
        if (lane == 63) sums[wave] = scan;
    }
    __syncthreads();
    if (t < GROUP_BINS) {
        int from = scan - v;
        for (int w = 0; w < wave; ++w) from += sums[w];
        next[t] = from;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t i = row0 + u * GROUP_THREADS + t;
        const int to = places(bin[u], i < n);
        if (i < n) perm[row0 + to] = (int32_t)i;
    }
}

// ---------------------------------------------------------------- t = s A x
// v as a sum of N values of T, rounded to nearest; all of an infinity or a NaN is in the first. (A finite v
// that would be rounded to infinity, next to the largest float: bf16's largest value first.)
template <class T, int N>
__device__ __forceinline__ void pieces_of(float v, T (&p)[N]) {
#pragma unroll
    for (int q = 0; q < N; ++q) {
        p[q] = (T)v;
        if (__is_same(T, __bf16) && fabsf((float)p[q]) == INFINITY && fabsf(v) < INFINITY) p[q] = (T)copysignf(0x1.fep127f, v);
        v = fabsf((float)p[q]) < INFINITY ? v - (float)p[q] : 0.0f;
    }
}

// What the projection reads of t. Few rows: f32, `f`, as FEW_PARTS parts to be added up. Tiles: as
// pieces of T for its matrix instructions, `plane` elements apart, whose sum is t: one in f32, three in bf16 (all
// 24 bits) and f16. f16: each row is scaled by a power of two to a largest value in [2^14, 2^15), undone by
// `back`; the sum of three is then t within half of f16's smallest step, 2^-25, which is 2^-39 of the largest.
// (Two pieces held 16 bits in bf16 and took within 1% of the time.)
constexpr int FEW_PARTS = 4;
template <class T>
constexpr int MID_PIECES = sizeof(T) == 2 ? 3 : 1;
template <class T>
struct Mid {
    float* f;
    T* piece;
    int64_t plane;
    float* back;
    int32_t* eff;  // few rows: a row's adapter and its rank, id * 256 + rank, -1 = none
    int ld;
};

// N values of a row from column c on, zeros past `in`
template <class T>
__device__ __forceinline__ typename Mma<T>::V row_piece(const T* row, int c, int in, bool whole) {
    if (whole || c + PIECE<T> <= in) return load_piece(row + c);
    typename Mma<T>::V v;
#pragma unroll
    for (int j = 0; j < PIECE<T>; ++j) v[j] = c + j < in ? row[c + j] : (T)0.0f;
    return v;
}

// Bound by the latency of its loads where rows are few: bf16 4096 x 4096, 64 rows: 26.5 us for the layer
// with one block a row tile, 22.8 with the sum in FEW_PARTS parts; by HBM where they are many.
// A block: 16 rows (of the permutation), the waves split the sum over `in`. Lays the rows out in
// fragment order (PACK) and computes t for them: the block's y-th, (y + gridDim.y)-th .. different
// adapter is its work; RT == 0: no adapters.
constexpr int SHRINK_WAVES = 8;
template <class T, int RT, bool SPLIT, bool PACK>
__global__ __launch_bounds__(64 * SHRINK_WAVES) void shrink_kernel(const T* __restrict__ x, int in, int64_t n,
                                                           const int32_t* __restrict__ perm, const T* __restrict__ a,
                                                           int64_t a_slot, int kt, const int32_t* __restrict__ ids,
                                                           const AdapterSlot* __restrict__ slot, int slots, Mid<T> t,
                                                           T* __restrict__ packed) {
    using V = typename Mma<T>::V;
    constexpr int N = PIECE<T>, R = RT ? RT : 1, WAVES = SHRINK_WAVES;
    __shared__ f32x4 red[RT ? WAVES : 1][R][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row0 = (int64_t)blockIdx.x * 16;
    const int64_t place = min(row0 + (lane & 15), n - 1);
    const int64_t my_row = perm ? perm[place] : place;
    const int mine = RT && lane < 16 && row0 + lane < n ? adapter_of(ids, slot, slots, my_row, n) : -1;
    if (RT && !SPLIT && blockIdx.y == 0 && blockIdx.z == 0 && threadIdx.x < 16 && row0 + lane < n)
        t.eff[row0 + lane] = mine < 0 ? -1 : mine * 256 + slot[mine].rank;
    unsigned long long todo = __ballot(mine >= 0);
    const T* xp = x + my_row * in;
    // several blocks may share the sum (gridDim.z): each then writes a part of t of its own
    const int parts = WAVES * gridDim.z, part = wave + WAVES * blockIdx.z;
    const int per = (kt / 2 + parts - 1) / parts * 2, k0 = min(kt, part * per), k1 = min(kt, k0 + per);
    const int whole = in / (2 * DEPTH<T>)*2;  // fragments without a zero
    T* to = packed + (int64_t)blockIdx.x * kt * (64 * N) + lane * N;
    bool pack = PACK && blockIdx.y == 0;
    for (int turn = 0; todo || pack; ++turn) {
        const int id = todo ? __builtin_amdgcn_readlane(mine, __ffsll(todo) - 1) : -1;
        todo &= ~__ballot(mine == id);
        const bool multiply = RT && id >= 0 && turn % gridDim.y == blockIdx.y;
        if (!multiply && !pack) continue;
        f32x4 acc[R] = {};
        const T* ap = a + (multiply ? id : 0) * a_slot + lane * N;
        auto sweep = [&](auto packs, auto multiplies) {
            constexpr bool PK = decltype(packs)::value, MU = decltype(multiplies)::value && RT > 0;
            constexpr int U = !MU || R <= 2 ? 8 : 16 / R;  // loads in flight, by registers
            int k = k0;
            for (; k + U <= min(k1, whole); k += U) {
                V xv[U], av[U][R];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    xv[u] = load_piece(xp + in_of<T>(k + u, lane >> 4));
                    if constexpr (MU)
#pragma unroll
                        for (int r = 0; r < R; ++r) av[u][r] = load_piece(ap + ((int64_t)r * kt + k + u) * (64 * N));
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if constexpr (PK) __builtin_memcpy(to + (int64_t)(k + u) * (64 * N), &xv[u], 16);
                    if constexpr (MU)
#pragma unroll
                        for (int r = 0; r < R; ++r) acc[r] = Mma<T>::run(av[u][r], xv[u], acc[r]);
                }
            }
            for (; k < k1; ++k) {
                const V xv = row_piece(xp, in_of<T>(k, lane >> 4), in, k < whole);
                if constexpr (PK) __builtin_memcpy(to + (int64_t)k * (64 * N), &xv, 16);
                if constexpr (MU)
#pragma unroll
                    for (int r = 0; r < R; ++r)
                        acc[r] = Mma<T>::run(load_piece(ap + ((int64_t)r * kt + k) * (64 * N)), xv, acc[r]);
            }
        };
        if (pack) sweep(std::integral_constant<bool, PACK>{}, std::true_type{});  // any adapter, where it has none
        else if constexpr (RT > 0) sweep(std::false_type{}, std::true_type{});
        pack = false;
        if (!multiply) continue;
        if constexpr (RT > 0) {
#pragma unroll
            for (int r = 0; r < RT; ++r) red[wave][r][lane] = acc[r];
            __syncthreads();
            if (wave == 0) {
                // lane l has ranks r * 16 + (l / 16) * 4 .. of row l % 16
                const AdapterSlot info = slot[id];
                auto value = [&](int r, float (&v)[4]) {
                    f32x4 sum = red[0][r][lane];
#pragma unroll
                    for (int w = 1; w < WAVES; ++w) sum += red[w][r][lane];
#pragma unroll
                    for (int j = 0; j < 4; ++j)  // past the adapter's rank: zeros, whatever x holds
                        v[j] = r * 16 + (lane >> 4) * 4 + j < info.rank ? sum[j] * info.scale : 0.0f;
                };
                const int64_t at = row0 + (lane & 15);  // the place in the permutation
                const bool own = __shfl(mine, lane & 15) == id;
                auto write = [&](int r, const float (&v)[4], float up) {
                    const int64_t o = at * t.ld + r * 16 + (lane >> 4) * 4;
                    if (!own) return;
                    if constexpr (!SPLIT) {
                        __builtin_memcpy(t.f + (int64_t)blockIdx.z * n * t.ld + o, v, 16);
                    } else {
                        T p[4][MID_PIECES<T>];
#pragma unroll
                        for (int j = 0; j < 4; ++j) pieces_of(v[j] * up, p[j]);
#pragma unroll
                        for (int q = 0; q < MID_PIECES<T>; ++q) {
                            const T four[4] = {p[0][q], p[1][q], p[2][q], p[3][q]};
                            __builtin_memcpy(t.piece + q * t.plane + o, four, sizeof(four));
                        }
                    }
                };
                if constexpr (SPLIT && __is_same(T, _Float16)) {
                    float v[RT][4], most = 0.0f;
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        value(r, v[r]);
#pragma unroll
                        for (int j = 0; j < 4; ++j)  // an infinity stays one, the others still have to fit
                            most = fmaxf(most, fabsf(v[r][j]) < INFINITY ? fabsf(v[r][j]) : 0.0f);
                    }
                    most = fmaxf(most, __shfl_xor(most, 16));
                    most = fmaxf(most, __shfl_xor(most, 32));
                    float up = 1.0f, down = 1.0f;
                    if (most > 0.0f) {
                        const int e = min(126, max(-126, 14 - ilogbf(most)));
                        up = ldexpf(1.0f, e), down = ldexpf(1.0f, -e);
                    }
                    if (own && lane < 16) t.back[at] = down;
#pragma unroll
                    for (int r = 0; r < RT; ++r) write(r, v[r], up);
                } else {
                    constexpr int TURNS = SPLIT && RT == 8 ? 1 : RT;  // (8 at once would spill)
#pragma unroll TURNS
                    for (int r = 0; r < RT; ++r) {
                        float v[4];
                        value(r, v);
                        write(r, v, 1.0f);
                    }
                }
                if (SPLIT && RT == 1 && t.ld > 16) {  // a fragment is 32 ranks deep
                    const float zero[4] = {};
                    write(1, zero, 1.0f);
                }
            }
            __syncthreads();
        }
    }
}

// ---------------------------------------------------------------- f32 as three bf16
// f32 products of many rows, as far as they fill the card, run on the bf16 matrix instructions, 16 times the f32 ones' rate: a value is
// exactly the sum of three bf16, h + m + l, each rounded to nearest from what the ones before leave:
// 8 bits each, |m| <= 2^-8 |h|, |l| <= 2^-17 |h|. Of the nine products the six largest are taken, h h, h m,
// m h, m m, h l and l h; the others are below 2^-24 |x w| together, half a step of an f32 product.
// bf16 has f32's range but for its smallest values, so each row of x and of W is scaled by a power of
// two to a largest value in [2^54, 2^55): a value down to 2^-165 of it is held exactly, smaller ones within
// 2^-189 of it, and the sum of 2^16 products stays in range. inv: 1 / scale. The three fragments of a depth are
// neighbours. inv is negative for a row with an infinity and no NaN: the product of an infinity and a part that
// is 0 would be a NaN, so its outputs are added up once more from the values themselves. One wave a row. 4096 x 4096, 2048 rows: 588 us with the f32 instructions, 337 so.
// (Two f16 values a number, three products: 206 us, but 22 bits of a row's largest values and fewer
// of its others, which an f32 layer cannot do with: x = (1, 1.23 2^-26 ..), W = (2^-40, 1.1 ..) was off by 2e-5.)
constexpr int SPLIT_PARTS = 3;
constexpr int SPLIT_EXP = 54;

template <bool WEIGHT>
__global__ __launch_bounds__(1024) void split_kernel(const float* __restrict__ x, int in, int64_t rows,
                                                    const int32_t* __restrict__ perm, int ktq,
                                                    __bf16* __restrict__ out, float* __restrict__ inv) {
    const int lane = threadIdx.x & 63, m = threadIdx.x >> 6;
    const int64_t place = WEIGHT ? out_of(blockIdx.x, m) : (int64_t)blockIdx.x * 16 + m;
    const bool there = place < rows;
    const float* row = x + (there ? perm ? perm[place] : place : 0) * in;
    auto piece = [&](int c, float (&v)[8]) {
        if (there && c + 8 <= in) __builtin_memcpy(v, row + c, 32);
        else
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = there && c + j < in ? row[c + j] : 0.0f;
    };
    float most = 0.0f;
    bool inf = false, nan = false;
    const int pieces = ktq * 4;
#pragma unroll 4
    for (int p = lane; p < pieces; p += 64) {
        float v[8];
        piece(p * 8, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            most = fmaxf(most, fabsf(v[j]) < INFINITY ? fabsf(v[j]) : 0.0f);
            inf |= fabsf(v[j]) == INFINITY, nan |= v[j] != v[j];
        }
    }
    inf = __any(inf) && !__any(nan);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));
    const int e = most > 0.0f ? min(126, SPLIT_EXP - ilogbf(most)) : 0;
    const float scale = ldexpf(1.0f, e);
    if (there && lane == 0) inv[place] = ldexpf(inf ? -1.0f : 1.0f, -e);
#pragma unroll 2
    for (int p = lane; p < pieces; p += 64) {
        float v[8];
        piece(p * 8, v);
        bf16x8 part[SPLIT_PARTS];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            __bf16 b[SPLIT_PARTS];
            pieces_of(v[j] * scale, b);
#pragma unroll
            for (int h = 0; h < SPLIT_PARTS; ++h) part[h][j] = b[h];
        }
        // the inverse of in_of: 8 pieces a pair of fragments, two by two of a lane
        const int q = (p >> 3) * 2 + (p & 1), to = ((p & 7) >> 1) * 16 + m;
        __bf16* o = out + ((int64_t)blockIdx.x * ktq + q) * SPLIT_PARTS * 512 + to * 8;
#pragma unroll
        for (int h = 0; h < SPLIT_PARTS; ++h) __builtin_memcpy(o + h * 512, &part[h], 16);
    }
}

// ---------------------------------------------------------------- few rows
// A block: a fragment tile's 16 outputs for all (<= 16 MT) rows; its waves split the sum and join in
// LDS. Bound by reading W once: bf16 4096 x 4096 10 us for 1 row, 14 for 16, 20.6 for 64, with t.
// As tiles (below): 33 rows 37 us to 19 here, 64 rows 36 to 21; f32 106 to 39; bf16 768 x
// 768, 64 rows 17 to 11.
constexpr int FEW_WAVES = 16;

// MT == 0: one row tile, x row-major.
template <class T, int MT0>
__global__ __launch_bounds__(64 * FEW_WAVES) void few_rows_kernel(const T* __restrict__ x, int in, int n,
                                                                 const T* __restrict__ w, int kt,
                                                                 const T* __restrict__ bias, const T* __restrict__ b,
                                                                 int64_t b_slot, int rk,
                                                                 const int32_t* __restrict__ eff,
                                                                 const float* __restrict__ t, int ldt, int out,
                                                                 T* __restrict__ y) {
    using V = typename Mma<T>::V;
    constexpr int N = PIECE<T>, MT = MT0 ? MT0 : 1;
    __shared__ f32x4 red[FEW_WAVES][MT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nt = blockIdx.x;
    // this thread's output: o = (row tile, row, output), one each (16 rows: of the first 256 threads)
    const int o = threadIdx.x, row = o >> 4, c = o & 15, col = out_of(nt, c);
    const bool there = o < MT * 256 && row < n && col < out;
    const int who = there && eff ? eff[row] : -1;
    const int per = (kt / 2 + FEW_WAVES - 1) / FEW_WAVES * 2, k0 = min(kt, wave * per), k1 = min(kt, k0 + per);
    const T* wp = w + (int64_t)nt * kt * (64 * N) + lane * N;
    const T* xp[MT];  // rows past n are not there: their lanes read the last one, or the last tile's
#pragma unroll
    for (int m = 0; m < MT; ++m)
        xp[m] = MT0 ? x + (int64_t)min(m, (n - 1) >> 4) * kt * (64 * N) + lane * N : x + (int64_t)min(lane & 15, n - 1) * in;
    const int whole = MT0 ? kt : in / (2 * DEPTH<T>)*2;
    auto piece = [&](int m, int k, bool all) -> V {
        if constexpr (MT0 > 0) return load_piece(xp[m] + (int64_t)k * (64 * N));
        else return row_piece(xp[m], in_of<T>(k, lane >> 4), in, all);
    };
    f32x4 acc[MT] = {};
    constexpr int U = MT == 4 ? 4 : 8;  // loads in flight, by registers
    int k = k0;
    for (; k + U <= min(k1, whole); k += U) {
        V wv[U], xv[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            wv[u] = load_piece(wp + (int64_t)(k + u) * (64 * N));
#pragma unroll
            for (int m = 0; m < MT; ++m) xv[u][m] = piece(m, k + u, true);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[m] = Mma<T>::run(wv[u], xv[u][m], acc[m]);
    }
#pragma unroll 2
    for (; k < k1; ++k) {
        const V wv = load_piece(wp + (int64_t)k * (64 * N));
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[m] = Mma<T>::run(wv, piece(m, k, k < whole), acc[m]);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) red[wave][m][lane] = acc[m];
    // B's row of this output: the piece of ranks p N .. is lane (p % 4) * 16 + c of fragment p / 4
    float d = 0.0f;
    if (who >= 0) {
        const int id = who >> 8, rank = who & 255;
        const T* bp = b + id * b_slot + (int64_t)nt * rk * (64 * N) + c * N;
        const float* tp = t + (int64_t)row * ldt;
        for (int p = 0; p * N < rank; ++p) {
            const V bv = load_piece(bp + ((p >> 2) * 64 + (p & 3) * 16) * N);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                float tv = tp[p * N + j];
#pragma unroll
                for (int q = 1; q < FEW_PARTS; ++q) tv += tp[(int64_t)q * n * ldt + p * N + j];
                d = fmaf(tv, (float)bv[j], d);
            }
        }
    }
    __syncthreads();
    if (!there) return;
    float v = 0.0f;
#pragma unroll
    for (int q = 0; q < FEW_WAVES; ++q) v += red[q][row >> 4][(c >> 2) * 16 + (row & 15)][c & 3];
    v += d;
    if (bias) v += (float)bias[col];
    y[(int64_t)row * out + col] = (T)v;
}

// ---------------------------------------------------------------- many rows
// A block: BM rows (of the permutation) x BN outputs; WM x WN waves; the sum in stages KF fragments
// deep, NS of which are in LDS or on their way to it (copied there without registers).
// KF == 1, large tiles: while a stage is multiplied from registers, the next one is read into others.
// Behind a stage's one barrier everybody has read it, so its place is free for stage s + NS, and has
// the next: the copies of NS - 2 stages more may still be on their way, which hides their latency.
// KF > 1, small tiles and split f32: a fragment is a few products only, so a barrier serves KF of them; behind it
// stage s has arrived and s - 1 is read, whose place the copies of s + NS - 1 take.
// Bound by LDS, which takes the copies and gives each fragment to WN or WM waves: about 200 bytes a ns
// of both whatever the tile; larger tiles need fewer for a product. Waves count too: a wave's copies
// go out about 100 ns apart, so the tiles of four waves of 64 x 64 and 128 x 64 were half as fast as of eight
// (bf16 4096 x 4096, 2048 rows: 110 and 107 us, 82 and 80 with eight).
template <int BM, int BN, int WM, int WN, int NS, int KF>
struct TileCfg {
    static constexpr int WAVES = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16;
    static constexpr int XF = BM / 16, WF = BN / 16;          // 1-KiB fragments of a stage
    static constexpr int XP = XF / WAVES, WP = WF / WAVES;    // copied by each wave, of each fragment's depth
    static constexpr int STAGE = (XF + WF) * KF * 1024;
    static_assert(XF % WAVES == 0 && WF % WAVES == 0 && TN % 2 == 0);
};

// All waves have read LDS as far as they asked for, and at most Vm of their copies are on their way.
// (Builtins, so that the compiler knows what has arrived.)
template <int Vm>
__device__ __forceinline__ void wait_and_meet() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt((Vm & 15) | (Vm >> 4) << 14 | 7 << 4);  // lgkmcnt 0
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
}

// The order of a half stage's instructions: one copy or one read of LDS between products, so that
// none of the three units waits for the others' turns.
template <int READS, int COPIES, int PRODUCTS>
__device__ __forceinline__ void spread() {
    constexpr int EACH = PRODUCTS / (READS + COPIES) > 0 ? PRODUCTS / (READS + COPIES) : 1;
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);
    }
#pragma unroll
    for (int i = 0; i < READS; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, PRODUCTS, 0);
}

// P: the products' type; __bf16 with T = float: a value's three fragments in turn, KF = 3.
template <class T, class P, int BM, int BN, int WM, int WN, int NS, int KF>
__global__ __launch_bounds__(64 * WM * WN) void tile_kernel(const P* __restrict__ x, const float* __restrict__ x_inv,
                                                           int64_t n, const P* __restrict__ w,
                                                           const float* __restrict__ w_inv, int kt, int nts,
                                                           const T* __restrict__ bias, const T* __restrict__ b,
                                                           int64_t b_slot, int rk, const int32_t* __restrict__ ids,
                                                           const int32_t* __restrict__ perm,
                                                           const AdapterSlot* __restrict__ slot, int slots, Mid<T> t,
                                                           int out, int tiles_m, int tiles_n, T* y,
                                                           const T* __restrict__ x_plain, const T* __restrict__ w_plain,
                                                           int in, int kt_plain) {  // (split f32)
    using Cf = TileCfg<BM, BN, WM, WN, NS, KF>;
    using V = typename Mma<T>::V;
    using PV = typename Mma<P>::V;
    constexpr bool SPLIT = !__is_same(T, P);
    static_assert(!SPLIT || KF == SPLIT_PARTS);
    constexpr int N = PIECE<T>, TM = Cf::TM, TN = Cf::TN;
    __shared__ __align__(16) unsigned char lds[NS * Cf::STAGE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave - wm * WN;
    // Blocks go to the 8 XCDs in turn: block i of XCD d is the i-th tile of the d-th part, so that an
    // L2 serves neighbouring tiles; in this order 8 tiles of rows share each tile of outputs.
    const int total = tiles_m * tiles_n;
    int tile = blockIdx.x;
    {
        const int part = (total + 7) / 8, d = tile & 7, i = tile >> 3;
        const int full = total - (part - 1) * 8;  // parts of the larger size
        tile = d < full ? d * part + i : full * part + (d - full) * (part - 1) + i;
    }
    const int band = tile / (8 * tiles_n), in_band = tile - band * 8 * tiles_n, rows_of_band = min(8, tiles_m - band * 8);
    const int tn = in_band / rows_of_band, tm = band * 8 + (in_band - tn * rows_of_band);
    const int64_t row0 = (int64_t)tm * BM;
    const int nt0 = tn * (BN / 16), ntw = nt0 + wn * TN;
    auto row_at = [&](int64_t place) -> int64_t {
        const int64_t p = min(place, n - 1);
        return perm ? perm[p] : p;
    };
    f32x4 acc[TM][TN];
    {
        constexpr int UNIT = 64 * PIECE<P>;  // elements of a fragment
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
        const P* xs[Cf::XP];
        const P* ws[Cf::WP];
#pragma unroll
        for (int j = 0; j < Cf::XP; ++j)
            xs[j] = x + min(row0 / 16 + wave * Cf::XP + j, (n - 1) / 16) * kt * UNIT;
#pragma unroll
        for (int j = 0; j < Cf::WP; ++j) ws[j] = w + (int64_t)min(nt0 + wave * Cf::WP + j, nts - 1) * kt * UNIT;
        // fragment k of the sum, the f-th of its stage: x's tiles, then W's
        auto copy = [&](int k, int buf, int f) {
            unsigned char* base = lds + buf * Cf::STAGE + f * (Cf::XF + Cf::WF) * 1024;
#pragma unroll
            for (int j = 0; j < Cf::XP; ++j)
                __builtin_amdgcn_global_load_lds(
                    (const void*)(xs[j] + (int64_t)k * UNIT + lane * PIECE<P>),
                    (__attribute__((address_space(3))) void*)(base + (wave * Cf::XP + j) * 1024), 16, 0, 0);
#pragma unroll
            for (int j = 0; j < Cf::WP; ++j)
                __builtin_amdgcn_global_load_lds(
                    (const void*)(ws[j] + (int64_t)k * UNIT + lane * PIECE<P>),
                    (__attribute__((address_space(3))) void*)(base + (Cf::XF + wave * Cf::WP + j) * 1024), 16, 0, 0);
        };
        auto fill = [&](int s, int buf) {  // past the end: copies of the last fragment, which nobody reads
#pragma unroll
            for (int f = 0; f < KF; ++f) copy(min(s * KF + f, kt - 1), buf, f);
        };
        PV xv[SPLIT ? 3 : 2][TM], wv[SPLIT ? 3 : 2][TN];
        auto read = [&](auto to, int buf, int f) {
            constexpr int h = decltype(to)::value;
            const unsigned char* base = lds + buf * Cf::STAGE + f * (Cf::XF + Cf::WF) * 1024 + lane * 16;
#pragma unroll
            for (int j = 0; j < TN; ++j) wv[h][j] = *(const PV*)(base + (Cf::XF + wn * TN + j) * 1024);
#pragma unroll
            for (int i = 0; i < TM; ++i) xv[h][i] = *(const PV*)(base + (wm * TM + i) * 1024);
        };
        auto multiply = [&](auto from, auto other) {
            constexpr int h = decltype(from)::value, o = decltype(other)::value;
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = Mma<P>::run(wv[h][j], xv[o][i], acc[i][j]);
        };
        constexpr int COPIES = Cf::XP + Cf::WP;
        using std::integral_constant;
        if constexpr (KF > 1) {
            const int stages = (kt + KF - 1) / KF;
#pragma unroll
            for (int s = 0; s < NS - 1; ++s) fill(s, s);  // as many as are counted below, there or not
            int buf = 0, last = NS - 1;
            for (int s = 0; s < stages; ++s) {
                wait_and_meet<(NS - 2) * COPIES * KF>();
                fill(s + NS - 1, last);
                constexpr integral_constant<int, 0> I0{};
                constexpr integral_constant<int, 1> I1{};
                constexpr integral_constant<int, 2> I2{};
                read(I0, buf, 0);
                if constexpr (SPLIT) {
                    read(I1, buf, 1);
                    multiply(I0, I0);
                    read(I2, buf, 2);
                    multiply(I0, I1);
                    multiply(I1, I0);
                    multiply(I1, I1);
                    multiply(I0, I2);
                    multiply(I2, I0);
                } else {
                    const int depth = min(KF, kt - s * KF);  // even
#pragma unroll
                    for (int f = 0; f < KF; f += 2) {
                        if (f >= depth) break;
                        read(I1, buf, f + 1);
                        multiply(I0, I0);
                        if (f + 2 < depth) read(I0, buf, f + 2);
                        multiply(I1, I1);
                    }
                }
                last = buf;
                buf = buf + 1 == NS ? 0 : buf + 1;
            }
            __builtin_amdgcn_s_waitcnt(0xf << 8 | 7 << 4);  // vmcnt 0: no copy outlives the loop
        } else {
            for (int s = 0; s < NS && s < kt; ++s) fill(s, s);
            wait_and_meet<0>();
            read(integral_constant<int, 0>{}, 0, 0);
            int s = 0, buf = 0;
            auto step = [&](auto at, bool full) {  // stage s is in registers, or on its way from LDS
                constexpr int h = decltype(at)::value;
                const int next = buf + 1 == NS ? 0 : buf + 1;
                if (full) {
                    wait_and_meet<(NS - 2) * COPIES>();
                    fill(s + NS, buf);
                    read(integral_constant<int, 1 - h>{}, next, 0);
                    multiply(at, at);
                    spread<TM + TN, COPIES, TM * TN>();
                    __builtin_amdgcn_sched_barrier(0);
                } else {
                    wait_and_meet<0>();
                    if (s + NS < kt) fill(s + NS, buf);
                    if (s + 1 < kt) read(integral_constant<int, 1 - h>{}, next, 0);
                    multiply(at, at);
                }
                buf = next;
                ++s;
            };
            for (; s + 1 + NS < kt;) {  // kt is even
                step(integral_constant<int, 0>{}, true);
                step(integral_constant<int, 1>{}, true);
            }
            for (; s < kt;) {
                step(integral_constant<int, 0>{}, false);
                step(integral_constant<int, 1>{}, false);
            }
        }
    }

    // y's pieces: lane l has outputs out_of(ntw + j, (l / 16) * 4 + r) of row l % 16 of tile i
    int64_t row[TM];
    int who[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int64_t place = row0 + (wm * TM + i) * 16 + (lane & 15);
        row[i] = row_at(place);
        who[i] = place < n ? adapter_of(ids, slot, slots, row[i], n) : -1;
        if (place >= n) row[i] = -1;
    }
    const int col0 = ntw * 16 + (lane >> 4) * 8;  // of the pair j, j + 1: col0 + j * 16 ..
    if constexpr (SPLIT) {
        bool infinite = false;
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const float x_scale = row[i] >= 0 ? x_inv[row0 + (wm * TM + i) * 16 + (lane & 15)] : 0.0f, xi = fabsf(x_scale);
            infinite |= x_scale < 0.0f;
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int col = col0 + (j >> 1) * 32 + (j & 1) * 4 + r;
                    // The scales' product can be past the largest float or below the smallest normal one where
                    // the result is neither: then one after the other, the larger first. (It is at least 1
                    // where the product is too large, at most 1 where it is too small, and a sum below
                    // 2^127: the first step ends in range unless the result does not.)
                    const float w_scale = col < out ? w_inv[col] : 0.0f, wi = fabsf(w_scale), s = xi * wi;
                    if (i == 0) infinite |= w_scale < 0.0f;
                    const bool normal = s >= 0x1p-126f && s < INFINITY;
                    acc[i][j][r] = normal ? acc[i][j][r] * s : acc[i][j][r] * fmaxf(xi, wi) * fminf(xi, wi);
                }
        }
        if (__any(infinite)) {
#pragma unroll 1
            for (int e = 0; e < TM * TN * 4; ++e) {
                const int ei = e / (TN * 4), ej = (e >> 2) % TN, er = e & 3;
                const int64_t place = row0 + (wm * TM + ei) * 16 + (lane & 15);
                const int col = col0 + (ej >> 1) * 32 + (ej & 1) * 4 + er;
                if (place >= n || col >= out || !(x_inv[place] < 0.0f || w_inv[col] < 0.0f)) continue;
                // the weights lie in fragment order: row m of tile nt
                const int nt = (col >> 5) * 2 + (col >> 2 & 1), m = (col >> 3 & 3) * 4 + (col & 3);
                const T* xr = x_plain + row_at(place) * in;
                const T* wr = w_plain + ((int64_t)nt * kt_plain * 64 + m) * N;
                float sum = 0.0f;
#pragma unroll 1
                for (int k = 0; k < in; ++k) {
                    const int f = (k / (2 * DEPTH<T>)) * 2 + (k / N & 1), piece = k / (2 * N) & 3;
                    sum = fmaf(xr[k], wr[((int64_t)f * 64 + piece * 16) * N + k % N], sum);
                }
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int j = 0; j < TN; ++j)
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[i][j][r] = e == (i * TN + j) * 4 + r ? sum : acc[i][j][r];
            }
        }
    }
    if (ids) {
        float back[TM];
#pragma unroll
        for (int i = 0; i < TM; ++i) back[i] = 1.0f;
        if constexpr (__is_same(T, _Float16))
#pragma unroll
            for (int i = 0; i < TM; ++i)
                if (who[i] >= 0) back[i] = t.back[row0 + (wm * TM + i) * 16 + (lane & 15)];
        for (int k = 0; k < rk; ++k) {
            int held = -1;
            V bv[TN];
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                // rows without an adapter hold anything: their products are dropped
                const int64_t place = min(row0 + (wm * TM + i) * 16 + (lane & 15), n - 1);
                const T* at = t.piece + place * t.ld + k * DEPTH<T> + (lane >> 4) * N;
                V tv[MID_PIECES<T>];
#pragma unroll
                for (int q = 0; q < MID_PIECES<T>; ++q) tv[q] = load_piece(at + q * t.plane);
                unsigned long long todo = __ballot(who[i] >= 0);
                while (todo) {
                    const int id = __builtin_amdgcn_readlane(who[i], __ffsll(todo) - 1);
                    todo &= ~__ballot(who[i] == id);
                    if (id != held) {
#pragma unroll
                        for (int j = 0; j < TN; ++j)
                            bv[j] = load_piece(b + id * b_slot + ((int64_t)min(ntw + j, nts - 1) * rk + k) * (64 * N) +
                                               lane * N);
                        held = id;
                    }
#pragma unroll
                    for (int j = 0; j < TN; ++j) {
                        f32x4 add{0, 0, 0, 0};
#pragma unroll
                        for (int q = 0; q < MID_PIECES<T>; ++q) add = Mma<T>::run(bv[j], tv[q], add);
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            acc[i][j][r] = who[i] == id ? fmaf(add[r], back[i], acc[i][j][r]) : acc[i][j][r];
                    }
                }
            }
        }
    }
#pragma unroll
    for (int j = 0; j < TN; j += 2) {
        const int col = col0 + j * 16;
        float bs[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) bs[r] = bias && col + r < out ? (float)bias[col + r] : 0.0f;
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            T v[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) v[r] = (T)(acc[i][j + (r >> 2)][r & 3] + bs[r]);
            T* o = y + row[i] * out + col;
            if (row[i] >= 0 && col + 8 <= out) __builtin_memcpy(o, v, sizeof(v));
            else if (row[i] >= 0)
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (col + r < out) o[r] = v[r];
        }
    }
}

}  // namespace

static int split_frags(int in) { return (in + 63) / 64 * 2; }  // 32 deep, an even number

AdapterShape adapter_shape(int32_t dtype, int32_t in, int32_t out, int32_t max_rank, int32_t slots) {
    const int piece = 16 / dtype_size(dtype), depth = 4 * piece;
    AdapterShape s{};
    s.dtype = dtype, s.in = in, s.out = out, s.slots = slots;
    s.kt = (in + 2 * depth - 1) / (2 * depth) * 2;
    s.nt = (out + 31) / 32 * 2;
    s.rt = (max_rank + 15) / 16;
    s.rt = s.rt <= 2 ? s.rt : s.rt <= 4 ? 4 : 8;  // the shrink kernel's forms
    s.rk = (max_rank + depth - 1) / depth;
    s.a_slot = (int64_t)s.rt * s.kt * 64 * piece;
    s.b_slot = (int64_t)s.nt * s.rk * 64 * piece;
    return s;
}

void adapter_pack(int32_t dtype, const void* src, int rows, int cols, int tiles, int frags, int what, void* dst) {
    with_dtype(dtype, [&](auto zero) {
        using T = decltype(zero);
        const int64_t pieces = (int64_t)tiles * frags * 64;
        RVX_LAUNCH("adapter_pack", pack_kernel<T>, dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, (const T*)src,
                   rows, cols, pieces, frags, what, (T*)dst);
    });
}

int64_t adapter_split_bytes(const AdapterShape& s) {
    return s.dtype == RVX_DTYPE_F32 ? (int64_t)s.nt * split_frags(s.in) * SPLIT_PARTS * 1024 : 0;
}
void adapter_split(const AdapterShape& s, const float* w, void* parts, float* inv) {
    RVX_LAUNCH("adapter_split", split_kernel<true>, dim3((unsigned)s.nt), dim3(1024), 0, w, s.in, (int64_t)s.out,
               (const int32_t*)nullptr, split_frags(s.in), (__bf16*)parts, inv);
}

void adapter_forward(const AdapterArgs& g) {
    const AdapterShape& s = g.s;
    // f32, up to 128 rows and long sums: twice the kernels for few rows, which read W once each. Whole layer, so and by
    // tiles: 4096 x 4096, 65 rows 58 and 106 us, 128: 74 and 105; 768 x 768 22 and 30, 28 and 30; 3000 x 100 41 and
    // 77, 57 and 77; three times, 160 rows: 768 x 768 39 and 30; short sums, 100 x 3000, 128 rows: 22 and 16.
    if (s.dtype == RVX_DTYPE_F32 && g.n > 64 && g.n <= 128 && s.in > 512) {
        for (int64_t r = 0; r < g.n; r += 64) {
            AdapterArgs part = g;
            part.n = std::min<int64_t>(64, g.n - r);
            part.x = (const float*)g.x + r * s.in;
            part.y = (float*)g.y + r * s.out;
            part.ids = g.ids ? g.ids + r : nullptr;
            adapter_forward(part);
        }
        return;
    }
    using std::integral_constant;
    with_dtype(s.dtype, [&](auto zero) {
        using T = decltype(zero);
        const T *x = (const T*)g.x, *w = (const T*)g.w, *bias = (const T*)g.bias, *b = (const T*)g.b;
        T* y = (T*)g.y;
        const int64_t n = g.n;
        const int cus = device().num_cus;
        const bool few = n <= 64;  // (as far as the registers of one block's rows go; figures at the kernel)
        Mid<T> t{};
        int32_t* perm = nullptr;
        if (g.ids) {
            t.ld = std::max(s.rk * DEPTH<T>, s.rt * 16);
            if (few) {
                t.f = scratch_f32("adapter_t", FEW_PARTS * n * t.ld + n);
                t.eff = (int32_t*)(t.f + FEW_PARTS * n * t.ld);
            } else {
                perm = (int32_t*)scratch_bytes("adapter_rows", n * 4);
                int bits = 1;
                while (bits < GROUP_BITS && (1 << bits) <= s.slots) ++bits;
                RVX_LAUNCH("adapter_group", group_rows_kernel, dim3((unsigned)((n + GROUP_ROWS - 1) / GROUP_ROWS)),
                           dim3(GROUP_THREADS), 0, g.ids, n, s.slots, bits, perm);
                t.plane = n * t.ld;
                t.piece = (T*)scratch_bytes("adapter_t", MID_PIECES<T> * t.plane * (int64_t)sizeof(T) + n * 4);
                t.back = __is_same(T, _Float16) ? (float*)(t.piece + MID_PIECES<T> * t.plane) : nullptr;
            }
        }
        constexpr bool F32 = __is_same(T, float);
        auto tiles = [&](int64_t bm, int64_t bn) { return (n + bm - 1) / bm * ((s.out + bn - 1) / bn); };
        auto rounds = [&](int64_t bm, int64_t bn) { return (tiles(bm, bn) + cus - 1) / cus; };
        const int64_t row_tiles = (n + 15) / 16;
        // without adapters one row tile is read as it is: its 16-row loads cost less than another launch
        // f32, the smaller tiles' f32 instructions where a tile a CU is all there is, or two with short sums: the split
        // and its launch cost more than six products at 16 times the rate save. Whole layer, f32 instructions and
        // split: 1024 x 1024, 300 rows 36 and 40 us, 1000: 41 and 46, 1300: 58 and 52; 4096 x 4096, 250 rows 107 and
        // 107, 320: 170 and 129; two tiles, 100 x 1000, 1500 rows 19 and 25; 768 x 768, 2048: 47 and 47.
        const bool split = F32 && !few && tiles(64, 64) > (s.in <= 512 ? 2 : 1) * (int64_t)cus;
        T* packed = split || (n <= 16 && !g.ids) ? nullptr : (T*)scratch_bytes("adapter_x", row_tiles * s.kt * 1024);
        // few row tiles: several blocks each, for the turns of different adapters and parts of the sum
        const unsigned spare = (unsigned)std::max<int64_t>(1, std::min<int64_t>(16, 2 * cus / row_tiles));
        const unsigned turns = g.ids ? few ? 16 : spare : 1, sums = few ? FEW_PARTS : g.ids ? 1 : std::min(spare, 4u);
        auto shrink = [&](auto rt, auto split, auto pack) {
            constexpr int RT = decltype(rt)::value;
            RVX_LAUNCH("adapter_shrink", (shrink_kernel<T, RT, decltype(split)::value, decltype(pack)::value>),
                       dim3((unsigned)row_tiles, turns, sums), dim3(64 * SHRINK_WAVES), 0, x, s.in, n, (const int32_t*)perm,
                       (const T*)g.a, s.a_slot, s.kt, g.ids, g.slot, s.slots, t, packed);
        };
        auto by_rank = [&](auto split, auto pack) {
            if (!g.ids) shrink(integral_constant<int, 0>{}, split, std::true_type{});
            else if (s.rt == 1) shrink(integral_constant<int, 1>{}, split, pack);
            else if (s.rt == 2) shrink(integral_constant<int, 2>{}, split, pack);
            else if (s.rt == 4) shrink(integral_constant<int, 4>{}, split, pack);
            else shrink(integral_constant<int, 8>{}, split, pack);
        };
        if (few) {
            if (packed) by_rank(std::false_type{}, std::true_type{});
        } else {
            if (packed) by_rank(std::true_type{}, std::true_type{});
            else if (g.ids) by_rank(std::true_type{}, std::false_type{});
        }
        if (few) {
            auto go = [&](auto mt) {
                constexpr int MT = decltype(mt)::value;
                RVX_LAUNCH("adapter_few_rows", (few_rows_kernel<T, MT>), dim3(s.nt), dim3(64 * FEW_WAVES), 0,
                           packed ? (const T*)packed : x, s.in, (int)n, w, s.kt, bias, b, s.b_slot, s.rk, (const int32_t*)t.eff, (const float*)t.f, t.ld, s.out, y);
            };
            if (!packed) go(integral_constant<int, 0>{});
            else if (n <= 16) go(integral_constant<int, 1>{});
            else if (n <= 32) go(integral_constant<int, 2>{});
            else go(integral_constant<int, 4>{});
            return;
        }
        auto go = [&](auto zero_p, const void* xp, const float* x_inv, const void* wp, int frags, auto bm, auto bn, auto wm,
                      auto wn, auto ns, auto kf) {
            using P = decltype(zero_p);
            constexpr int BM = decltype(bm)::value, BN = decltype(bn)::value, WM = decltype(wm)::value,
                          WN = decltype(wn)::value, NS = decltype(ns)::value;
            const int tm = (int)((n + BM - 1) / BM), tn = (s.out + BN - 1) / BN;
            RVX_LAUNCH("adapter_tile", (tile_kernel<T, P, BM, BN, WM, WN, NS, decltype(kf)::value>), dim3((unsigned)(tm * tn)),
                       dim3(64 * WM * WN), 0, (const P*)xp, x_inv, n, (const P*)wp, g.w_inv, frags, s.nt, bias, b, s.b_slot,
                       s.rk, g.ids, (const int32_t*)perm, g.slot, s.slots, t, s.out, tm, tn, y, x, w, s.in, s.kt);
        };
        constexpr integral_constant<int, 1> I1{};
        constexpr integral_constant<int, 2> I2{};
        constexpr integral_constant<int, 3> I3{};
        constexpr integral_constant<int, 4> I4{};
        constexpr integral_constant<int, 64> I64{};
        constexpr integral_constant<int, 128> I128{};
        constexpr integral_constant<int, 256> I256{};
        if (!split) {
            if constexpr (F32) return go(T{}, packed, nullptr, w, s.kt, I64, I64, I2, I2, I4, I2);
        }
        if constexpr (F32) {
            const int ktq = split_frags(s.in);
            const int64_t bytes = row_tiles * ktq * SPLIT_PARTS * 1024;
            auto* parts = (char*)scratch_bytes("adapter_x", bytes + n * 4);
            auto* x_inv = (float*)(parts + bytes);
            RVX_LAUNCH("adapter_split", split_kernel<false>, dim3((unsigned)row_tiles), dim3(1024), 0, x, s.in, n,
                       (const int32_t*)perm, ktq, (__bf16*)parts, x_inv);
            // whole layer, 4096 x 4096: 512 rows 141 us by 64 x 64, 178 by 128 x 128; 1024: 242, 208 and 288 by
            // 256 x 128; 2048: 428, 365, 337; 4096: 847, 707, 654. A round of the larger tiles takes 7 / 4 of one of the
            // smaller.
            if (tiles(128, 128) < cus) go(__bf16{}, parts, x_inv, g.w_split, SPLIT_PARTS * ktq, I64, I64, I2, I2, I3, I3);
            else if (7 * rounds(256, 128) <= 4 * rounds(128, 128))
                go(__bf16{}, parts, x_inv, g.w_split, SPLIT_PARTS * ktq, I256, I128, I4, I2, I2, I3);
            else go(__bf16{}, parts, x_inv, g.w_split, SPLIT_PARTS * ktq, I128, I128, I4, I2, I3, I3);
        } else {
            // whole layer, bf16 4096 x 4096: 512 rows 43 us by 64 x 64, 48 by 128 x 128, 66 by 256 x 128, 106 by 256
            // x 256; 1024: 69, 53, 67, 106; 2048: 120, 83, 79, 109; 4096: 227, 152, 149, 135; 8192: 432, 286, 280, 253.
            // A round of the largest takes 7 / 4 of one of 256 x 128; two tiles of 128 x 128 on a CU as long as one
            // of these.
            if (tiles(128, 128) < cus) go(T{}, packed, nullptr, w, s.kt, I64, I64, I2, I2, I4, I2);
            else if (8 * tiles(256, 128) <= 5 * cus) go(T{}, packed, nullptr, w, s.kt, I128, I128, I4, I2, I4, I1);
            else if (7 * rounds(256, 256) <= 4 * rounds(256, 128)) go(T{}, packed, nullptr, w, s.kt, I256, I256, I2, I4, I4, I1);
            else go(T{}, packed, nullptr, w, s.kt, I256, I128, I4, I2, I4, I1);
        }
    });
}

}  // namespace rvx
