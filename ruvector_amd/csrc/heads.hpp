// heads.hpp — what the typed operators around the graph layers share: element types, their
// vector loads and stores, argument checks, and the launch wrappers of k_embedding.hip,
// k_logprobs.hip and k_adapter.hip.
#pragma once
#include "common.hpp"
#include "graph.hpp"

namespace rvx {

// ---- element types -------------------------------------------------------
inline int dtype_size(int32_t dtype) { return dtype == RVX_DTYPE_F32 ? 4 : 2; }

template <class F>
void with_dtype(int32_t dtype, F&& f) {  // f(T{}) for the element type T of `dtype` (checked before)
    if (dtype == RVX_DTYPE_F32) f(float{});
    else if (dtype == RVX_DTYPE_F16) f(_Float16{});
    else f(__bf16{});
}

// 16 bytes of T at any element address: rows of an odd width start at odd elements, and gfx950
// takes vector loads and stores at any address.
// (A vector type: arrays of 16-bit values would be spread over a register each.)
template <class T>
struct Vec16 {
    static constexpr int N = 16 / (int)sizeof(T);
    T v __attribute__((ext_vector_type(N)));
};
template <class T>
__device__ __forceinline__ Vec16<T> load16(const T* p) {
    Vec16<T> r;
    __builtin_memcpy(&r, p, 16);
    return r;
}
template <class T>
__device__ __forceinline__ void store16(T* p, const Vec16<T>& r) {
    __builtin_memcpy(p, &r, 16);
}

// Between a wave's write and its lanes' reads of LDS: a wave's LDS instructions run in their order, so
// only the compiler has to keep it. (A fence would also wait for every load on its way.)
__device__ __forceinline__ void wave_lds_order() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
}

// ---- argument checks -----------------------------------------------------
inline void check_dtype(int32_t dtype) {
    RVX_REQUIRE(dtype >= RVX_DTYPE_F32 && dtype <= RVX_DTYPE_BF16, RVX_ERR_INVALID_PARAMETER,
                "unknown dtype " + std::to_string(dtype));
}
// `buf` holds rows of `ld` elements of `size` bytes, the last one `width` long, on the current device
inline void check_rows(const rvx_buffer* buf, const char* what, int64_t rows, int64_t width, int64_t ld, int size) {
    RVX_REQUIRE(buf, RVX_ERR_INVALID_PARAMETER, std::string("null ") + what);
    const __int128 need = rows > 0 ? ((__int128)(rows - 1) * ld + width) * size : 0;
    RVX_REQUIRE(buf->mem.bytes >= need, RVX_ERR_DIMENSION_MISMATCH,
                std::string(what) + " holds " + std::to_string(buf->mem.bytes) + " bytes, " +
                    std::to_string(rows) + " x " + std::to_string(ld) + " values need more");
    RVX_REQUIRE(!buf->mem.p || buf->mem.dev == device().id, RVX_ERR_INVALID_PARAMETER,
                std::string(what) + " is on device " + std::to_string(buf->mem.dev) + ", not the current one");
}
inline void check_apart(const rvx_buffer* a, const rvx_buffer* b, const char* what) {
    RVX_REQUIRE(!a || !b || a != b, RVX_ERR_INVALID_PARAMETER, std::string(what) + " must be different buffers");
}

// ---- rows of a table by id (k_embedding.hip) -----------------------------
constexpr int EMBED_MAX_DIM = 1 << 16;
void embedding_forward(int32_t dtype, const void* table, int64_t rows, int dim, const int64_t* ids, int64_t n,
                       float scale, void* out);
void embedding_backward(int32_t dtype, const void* grad_out, const int64_t* ids, int64_t n, int64_t rows, int dim,
                        float scale, bool accumulate, int32_t table_dtype, void* grad_table);

// ---- log probabilities over rows of scores (k_logprobs.hip) --------------
constexpr int LOGPROBS_MAX_K = 64;
struct LogProbsOut {  // null = not wanted
    float* logp; int64_t* rank; float* entropy; float* stats; int64_t* top_ids; float* top_logp;
};
void log_probs(int32_t dtype, const void* scores, int64_t n, int64_t c, int64_t ld, float temperature,
               const int64_t* targets, int k, const LogProbsOut& out);
void log_probs_backward(int32_t dtype, const void* scores, int64_t n, int64_t c, int64_t ld, float temperature,
                        const int64_t* targets, const float* stats, const float* grad_logp, const float* entropy,
                        const float* grad_entropy, void* grad, int64_t ld_grad);

}  // namespace rvx
