// k_adapter.hip — y_i = W x_i + bias + s_r B_r (A_r x_i) with r = ids[i], the adapter of row i.
//
// Two launches: t_i = s_r A_r x_i for every row (f32, n x rank), then the projection whose
// epilogue adds B_r t_i. Rows may come in any order of adapters: each 16-row tile goes over the
// different adapters among its rows, so rows of one request cost one turn and a tile of 16
// requests reads 16 adapters, which are all needed.
//
// Weights lie in fragment order: the 16 rows x 64 bytes that one matrix instruction takes from
// one operand are 1 KiB, lane l's 16 bytes at l * 16 (row l % 16, elements (l / 16) * N ..). A
// wave loads a fragment with one coalesced instruction, copies it to LDS as it is, and reads it
// back without bank conflicts.
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
template <class T>
__global__ __launch_bounds__(256) void pack_kernel(const T* __restrict__ src, int rows, int cols, int64_t pieces,
                                                  int frags, T* __restrict__ dst) {
    constexpr int N = PIECE<T>;
    const int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (p >= pieces) return;
    const int lane = (int)(p & 63);
    const int64_t f = p >> 6;
    const int row = (int)(f / frags) * 16 + (lane & 15);
    const int col = (int)(f % frags) * DEPTH<T> + (lane >> 4) * N;
    T v[N];
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = row < rows && col + j < cols ? src[(int64_t)row * cols + col + j] : (T)0.0f;
    __builtin_memcpy(dst + p * N, v, 16);
}

// rows of x with zeros behind them, up to whole pairs of fragments
template <class T>
__global__ __launch_bounds__(256) void pad_kernel(const T* __restrict__ x, int64_t n, int in, int ld, T* __restrict__ out) {
    const int64_t total = n * ld;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / ld;
        const int c = (int)(i - r * ld);
        out[i] = c < in ? x[r * in + c] : (T)0.0f;
    }
}

__device__ __forceinline__ int adapter_of(const int32_t* ids, const AdapterSlot* slot, int slots, int64_t row, int64_t n) {
    if (!ids || row >= n) return -1;
    const int id = ids[row];
    return id >= 0 && id < slots && slot[id].rank > 0 ? id : -1;
}

// ---------------------------------------------------------------- t = s A x
constexpr int SH_WAVES = 8;

// A block: 16 * SM rows, the waves split the sum over `in`. The block's y-th, (y + gridDim.y)-th
// .. different adapter is its work.
template <class T, int SM, int RT>
__global__ __launch_bounds__(64 * SH_WAVES) void shrink_kernel(const T* __restrict__ x, int ldx, int64_t n,
                                                              const T* __restrict__ a, int64_t a_slot, int kt,
                                                              const int32_t* __restrict__ ids,
                                                              const AdapterSlot* __restrict__ slot, int slots,
                                                              float* __restrict__ t, int ldt) {
    using V = typename Mma<T>::V;
    constexpr int N = PIECE<T>;
    __shared__ f32x4 red[SH_WAVES][SM * RT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row0 = (int64_t)blockIdx.x * (16 * SM);
    const int mine = lane < 16 * SM ? adapter_of(ids, slot, slots, row0 + lane, n) : -1;
    unsigned long long todo = __ballot(mine >= 0);
    const T* xp[SM];
#pragma unroll
    for (int m = 0; m < SM; ++m)
        xp[m] = x + min(row0 + m * 16 + (lane & 15), n - 1) * ldx + (lane >> 4) * N;
    const int per = (kt + SH_WAVES - 1) / SH_WAVES, k0 = min(kt, wave * per), k1 = min(kt, k0 + per);
    for (int turn = 0; todo; ++turn) {
        const int id = __builtin_amdgcn_readlane(mine, __ffsll(todo) - 1);
        todo &= ~__ballot(mine == id);
        if (turn % gridDim.y != blockIdx.y) continue;
        f32x4 acc[SM][RT] = {};
        const T* ap = a + id * a_slot + lane * N;
#pragma unroll 4
        for (int k = k0; k < k1; ++k) {
            V xv[SM];
#pragma unroll
            for (int m = 0; m < SM; ++m) xv[m] = load_piece(xp[m] + k * DEPTH<T>);
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const V av = load_piece(ap + ((int64_t)r * kt + k) * (64 * N));
#pragma unroll
                for (int m = 0; m < SM; ++m) acc[m][r] = Mma<T>::run(xv[m], av, acc[m][r]);
            }
        }
#pragma unroll
        for (int m = 0; m < SM; ++m)
#pragma unroll
            for (int r = 0; r < RT; ++r) red[wave][m * RT + r][lane] = acc[m][r];
        __syncthreads();
        const AdapterSlot info = slot[id];
        for (int i = wave; i < SM * RT; i += SH_WAVES) {
            f32x4 s = red[0][i][lane];
#pragma unroll
            for (int w = 1; w < SH_WAVES; ++w) s += red[w][i][lane];
            const int m = i / RT, r = i - m * RT;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t row = row0 + m * 16 + (lane >> 4) * 4 + j;
                const int c = r * 16 + (lane & 15);  // past the adapter's rank: zeros, whatever x holds
                if (adapter_of(ids, slot, slots, row, n) == id) t[row * ldt + c] = c < info.rank ? s[j] * info.scale : 0.0f;
            }
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- few rows
// A block: 16 columns of y for all (<= 16 MT) rows; its waves split the sum and join in LDS. Bound
// by reading W once.
constexpr int FEW_WAVES = 8;

template <class T, int MT>
__global__ __launch_bounds__(64 * FEW_WAVES) void few_rows_kernel(const T* __restrict__ x, int ldx, int n,
                                                                 const T* __restrict__ w, int kt,
                                                                 const T* __restrict__ bias, const T* __restrict__ b,
                                                                 int64_t b_slot, int rk,
                                                                 const int32_t* __restrict__ ids,
                                                                 const AdapterSlot* __restrict__ slot, int slots,
                                                                 const float* __restrict__ t, int ldt, int out,
                                                                 T* __restrict__ y) {
    using V = typename Mma<T>::V;
    constexpr int N = PIECE<T>;
    __shared__ f32x4 red[FEW_WAVES][MT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nt = blockIdx.x;
    const int per = (kt + FEW_WAVES - 1) / FEW_WAVES, k0 = min(kt, wave * per), k1 = min(kt, k0 + per);
    const T* wp = w + (int64_t)nt * kt * (64 * N) + lane * N;
    const T* xp[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) xp[m] = x + (int64_t)min(m * 16 + (lane & 15), n - 1) * ldx + (lane >> 4) * N;
    f32x4 acc[MT] = {};
#pragma unroll 4
    for (int k = k0; k < k1; ++k) {
        const V wv = load_piece(wp + (int64_t)k * (64 * N));
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[m] = Mma<T>::run(load_piece(xp[m] + k * DEPTH<T>), wv, acc[m]);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) red[wave][m][lane] = acc[m];
    __syncthreads();
    for (int o = threadIdx.x; o < MT * 256; o += 64 * FEW_WAVES) {
        const int m = o >> 8, row = m * 16 + (o >> 4 & 15), c = o & 15, col = nt * 16 + c;
        if (row >= n || col >= out) continue;
        float v = 0.0f;
#pragma unroll
        for (int q = 0; q < FEW_WAVES; ++q) v += red[q][m][(o >> 6 & 3) * 16 + c][o >> 4 & 3];
        const int id = adapter_of(ids, slot, slots, row, n);
        if (id >= 0) {
            // B's row `col`: the piece of ranks 8 p .. (f32: 4 p ..) is lane (p % 4) * 16 + c of fragment p / 4
            const T* bp = b + id * b_slot + (int64_t)nt * rk * (64 * N) + c * N;
            const float* tp = t + (int64_t)row * ldt;
            const int pieces = (slot[id].rank + N - 1) / N;
            float d = 0.0f;
            for (int p = 0; p < pieces; ++p) {
                const V bv = load_piece(bp + ((p >> 2) * 64 + (p & 3) * 16) * N);
#pragma unroll
                for (int j = 0; j < N; ++j) d = fmaf(tp[p * N + j], (float)bv[j], d);
            }
            v += d;
        }
        if (bias) v += (float)bias[col];
        y[(int64_t)row * out + col] = (T)v;
    }
}

// ---------------------------------------------------------------- many rows
// The epilogue takes t's rows as fragments of T, hi + lo: 16 (bf16) or 22 (f16) bits of each
// value, so that t's rounding is far below y's. f16: the row is first scaled by a power of two
// to below 2^15 (t may be larger than f16 holds); `back` undoes it.
template <class T, int BM, int BN, int WM, int WN>
struct TileCfg {
    static constexpr int WAVES = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16;
    static constexpr int FRAGS = (BM + BN) / 16 * 2;  // 1-KiB pieces of a stage: 2 fragments deep
    static constexpr int STAGE = FRAGS * 1024;
    static_assert(FRAGS % WAVES == 0);
};

template <class T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void tile_kernel(const T* __restrict__ x, int ldx, int64_t n,
                                                           const T* __restrict__ w, int kt, int nts,
                                                           const T* __restrict__ bias, const T* __restrict__ b,
                                                           int64_t b_slot, int rk, const int32_t* __restrict__ ids,
                                                           const AdapterSlot* __restrict__ slot, int slots,
                                                           const float* __restrict__ t, int ldt, int tw, int out,
                                                           int tiles_m, int tiles_n, T* __restrict__ y) {
    using Cf = TileCfg<T, BM, BN, WM, WN>;
    using V = typename Mma<T>::V;
    constexpr int N = PIECE<T>, TM = Cf::TM, TN = Cf::TN, PER = Cf::FRAGS / Cf::WAVES, A_FRAGS = BM / 16 * 2;
    __shared__ __align__(16) unsigned char lds[2 * Cf::STAGE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave - wm * WN;
    // Blocks go to the 8 XCDs in turn: block i of XCD d is tile (d, i) of a cut into 8 parts, so
    // that an L2 serves neighbouring tiles.
    const int total = tiles_m * tiles_n;
    int tile = blockIdx.x;
    {
        const int part = (total + 7) / 8, d = tile & 7, i = tile >> 3;
        const int full = total - (part - 1) * 8;  // parts of the larger size
        tile = d < full ? d * part + i : full * part + (d - full) * (part - 1) + i;
    }
    const int tm = tile / tiles_n, tn = tile - tm * tiles_n;
    const int64_t row0 = (int64_t)tm * BM;
    const int nt0 = tn * (BN / 16);

    // this wave's pieces of a stage: fragments f = wave * PER + j; first those of x, then W's
    const T* src[PER];
    int step[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int f = wave * PER + j;
        if (f < A_FRAGS) {
            const int64_t row = min(row0 + (f >> 1) * 16 + (lane & 15), n - 1);
            src[j] = x + row * ldx + (f & 1) * DEPTH<T> + (lane >> 4) * N;
            step[j] = 2 * DEPTH<T>;
        } else {
            const int g = f - A_FRAGS;
            const int nt = min(nt0 + (g >> 1), nts - 1);
            src[j] = w + ((int64_t)nt * kt + (g & 1)) * (64 * N) + lane * N;
            step[j] = 2 * 64 * N;
        }
    }
    auto fill = [&](int s, int buf) {
#pragma unroll
        for (int j = 0; j < PER; ++j)
            __builtin_amdgcn_global_load_lds(
                (const void*)(src[j] + (int64_t)s * step[j]),
                (__attribute__((address_space(3))) void*)(lds + buf * Cf::STAGE + (wave * PER + j) * 1024), 16, 0, 0);
    };
    f32x4 acc[TM][TN] = {};
    const int stages = kt / 2;
    fill(0, 0);
    for (int s = 0; s < stages; ++s) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();  // stage s is there, and everybody has read stage s - 1
        if (s + 1 < stages) fill(s + 1, (s + 1) & 1);
        const unsigned char* base = lds + (s & 1) * Cf::STAGE;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            V av[TM], bv[TN];
#pragma unroll
            for (int i = 0; i < TM; ++i) av[i] = *(const V*)(base + ((wm * TM + i) * 2 + h) * 1024 + lane * 16);
#pragma unroll
            for (int i = 0; i < TN; ++i) bv[i] = *(const V*)(base + (A_FRAGS + (wn * TN + i) * 2 + h) * 1024 + lane * 16);
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = Mma<T>::run(av[i], bv[j], acc[i][j]);
        }
    }

    const int ntw = nt0 + wn * TN;
    if (ids) {
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const int64_t r0 = row0 + (wm * TM + i) * 16;
            const int mine = lane < 16 ? adapter_of(ids, slot, slots, r0 + lane, n) : -1;
            unsigned long long todo = __ballot(mine >= 0);
            int at[4];  // the adapters of this lane's four rows of C
#pragma unroll
            for (int r = 0; r < 4; ++r) at[r] = __shfl(mine, (lane >> 4) * 4 + r);
            while (todo) {
                const int id = __builtin_amdgcn_readlane(mine, __ffsll(todo) - 1);
                todo &= ~__ballot(mine == id);
                f32x4 add[TN] = {};
                float back[4] = {1.0f, 1.0f, 1.0f, 1.0f};
                // rows of other adapters give products that are dropped below
                const float* tp = t + min(r0 + (lane & 15), n - 1) * ldt + (lane >> 4) * N;
                float up = 1.0f;
                if constexpr (sizeof(T) == 2 && !__is_same(T, __bf16)) {
                    float m = 0.0f;
                    for (int k = 0; k < rk; ++k)
#pragma unroll
                        for (int j = 0; j < N; ++j)
                            m = fmaxf(m, k * DEPTH<T> + (lane >> 4) * N < tw ? fabsf(tp[k * DEPTH<T> + j]) : 0.0f);
                    m = fmaxf(m, __shfl_xor(m, 16));
                    m = fmaxf(m, __shfl_xor(m, 32));
                    const int e = m > 0.0f && m < INFINITY ? min(126, max(-126, 14 - ilogbf(m))) : 0;
                    up = ldexpf(1.0f, e);
                    const float down = ldexpf(1.0f, -e);
#pragma unroll
                    for (int r = 0; r < 4; ++r) back[r] = __shfl(down, (lane >> 4) * 4 + r);
                }
                for (int k = 0; k < rk; ++k) {
                    V hi, lo;
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        const float v = k * DEPTH<T> + (lane >> 4) * N < tw ? tp[k * DEPTH<T> + j] * up : 0.0f;
                        hi[j] = (T)v;
                        lo[j] = (T)(v - (float)hi[j]);
                    }
#pragma unroll
                    for (int j = 0; j < TN; ++j) {
                        const int nt = min(ntw + j, nts - 1);
                        const V bv = load_piece(b + id * b_slot + ((int64_t)nt * rk + k) * (64 * N) + lane * N);
                        add[j] = Mma<T>::run(hi, bv, add[j]);
                        if constexpr (sizeof(T) == 2) add[j] = Mma<T>::run(lo, bv, add[j]);
                    }
                }
#pragma unroll
                for (int j = 0; j < TN; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (at[r] == id) acc[i][j][r] = fmaf(add[j][r], back[r], acc[i][j][r]);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < TN; ++j) {
        const int col = (ntw + j) * 16 + (lane & 15);
        if (col >= out) continue;
        const float bs = bias ? (float)bias[col] : 0.0f;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int64_t row = row0 + (wm * TM + i) * 16 + (lane >> 4) * 4 + r;
                if (row < n) y[row * out + col] = (T)(acc[i][j][r] + bs);
            }
    }
}

}  // namespace

AdapterShape adapter_shape(int32_t dtype, int32_t in, int32_t out, int32_t max_rank, int32_t slots) {
    const int piece = 16 / dtype_size(dtype), depth = 4 * piece;
    AdapterShape s{};
    s.dtype = dtype, s.in = in, s.out = out, s.slots = slots;
    s.kt = (in + 2 * depth - 1) / (2 * depth) * 2;
    s.nt = (out + 15) / 16;
    s.rt = (max_rank + 15) / 16;
    s.rt = s.rt <= 2 ? s.rt : s.rt <= 4 ? 4 : 8;  // the shrink kernel's forms
    s.rk = (max_rank + depth - 1) / depth;
    s.a_slot = (int64_t)s.rt * s.kt * 64 * piece;
    s.b_slot = (int64_t)s.nt * s.rk * 64 * piece;
    return s;
}

void adapter_pack(int32_t dtype, const void* src, int rows, int cols, int tiles, int frags, void* dst) {
    with_dtype(dtype, [&](auto zero) {
        using T = decltype(zero);
        const int64_t pieces = (int64_t)tiles * frags * 64;
        RVX_LAUNCH("adapter_pack", pack_kernel<T>, dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, (const T*)src,
                   rows, cols, pieces, frags, (T*)dst);
    });
}

void adapter_forward(const AdapterArgs& g) {
    const AdapterShape& s = g.s;
    with_dtype(s.dtype, [&](auto zero) {
        using T = decltype(zero);
        const T *x = (const T*)g.x, *w = (const T*)g.w, *bias = (const T*)g.bias, *b = (const T*)g.b;
        T* y = (T*)g.y;
        const int64_t n = g.n;
        const int cus = device().num_cus;
        int ldx = s.in;
        if (s.in != s.kt * DEPTH<T>) {
            ldx = s.kt * DEPTH<T>;
            T* padded = (T*)scratch_bytes("adapter_x", n * ldx * (int64_t)sizeof(T));
            RVX_LAUNCH("adapter_pad", pad_kernel<T>, dim3((unsigned)std::min<int64_t>((n * ldx + 255) / 256, 16LL * cus)),
                       dim3(256), 0, x, n, s.in, ldx, padded);
            x = padded;
        }
        const int ldt = std::max(s.rk * DEPTH<T>, s.rt * 16);
        float* t = nullptr;
        if (g.ids) {
            t = scratch_f32("adapter_t", n * ldt);
            auto go = [&](auto sm, auto rt) {
                constexpr int SM = decltype(sm)::value, RT = decltype(rt)::value;
                const unsigned tiles = (unsigned)((n + 16 * SM - 1) / (16 * SM));
                const unsigned turns = SM == 1 ? 16 : 1;
                RVX_LAUNCH("adapter_shrink", (shrink_kernel<T, SM, RT>), dim3(tiles, turns), dim3(64 * SH_WAVES), 0, x, ldx,
                           n, (const T*)g.a, s.a_slot, s.kt, g.ids, g.slot, s.slots, t, ldt);
            };
            auto by_rank = [&](auto sm) {
                if (s.rt == 1) go(sm, std::integral_constant<int, 1>{});
                else if (s.rt == 2) go(sm, std::integral_constant<int, 2>{});
                else if (s.rt == 4) go(sm, std::integral_constant<int, 4>{});
                else go(sm, std::integral_constant<int, 8>{});
            };
            if (n <= 1024) by_rank(std::integral_constant<int, 1>{});
            else by_rank(std::integral_constant<int, 2>{});
        }
        if (n <= 64) {
            auto go = [&](auto mt) {
                constexpr int MT = decltype(mt)::value;
                RVX_LAUNCH("adapter_few_rows", (few_rows_kernel<T, MT>), dim3(s.nt), dim3(64 * FEW_WAVES), 0, x, ldx, (int)n,
                           w, s.kt, bias, b, s.b_slot, s.rk, g.ids, g.slot, s.slots, (const float*)t, ldt, s.out, y);
            };
            if (n <= 16) go(std::integral_constant<int, 1>{});
            else if (n <= 32) go(std::integral_constant<int, 2>{});
            else go(std::integral_constant<int, 4>{});
            return;
        }
        auto go = [&](auto bm, auto bn, auto wm, auto wn) {
            constexpr int BM = decltype(bm)::value, BN = decltype(bn)::value, WM = decltype(wm)::value, WN = decltype(wn)::value;
            const int tm = (int)((n + BM - 1) / BM), tn = (s.out + BN - 1) / BN;
            RVX_LAUNCH("adapter_tile", (tile_kernel<T, BM, BN, WM, WN>), dim3((unsigned)(tm * tn)), dim3(64 * WM * WN), 0, x,
                       ldx, n, w, s.kt, s.nt, bias, b, s.b_slot, s.rk, g.ids, g.slot, s.slots, (const float*)t, ldt,
                       s.rt * 16, s.out, tm, tn, y);
        };
        using std::integral_constant;
        auto tiles = [&](int64_t bm, int64_t bn) { return (n + bm - 1) / bm * ((s.out + bn - 1) / bn); };
        if (tiles(256, 256) >= cus)
            go(integral_constant<int, 256>{}, integral_constant<int, 256>{}, integral_constant<int, 2>{}, integral_constant<int, 4>{});
        else if (tiles(128, 128) >= cus)
            go(integral_constant<int, 128>{}, integral_constant<int, 128>{}, integral_constant<int, 2>{}, integral_constant<int, 2>{});
        else
            go(integral_constant<int, 64>{}, integral_constant<int, 64>{}, integral_constant<int, 2>{}, integral_constant<int, 2>{});
    });
}

}  // namespace rvx
