// adapter.hpp — AdapterLinear: a shared projection with one low-rank adapter per row
// (k_adapter.hip: kernels and launches; api_adapter.cpp: the C ABI).
#pragma once
#include "heads.hpp"

namespace rvx {

constexpr int ADAPTER_MAX_RANK = 128;
constexpr int ADAPTER_MAX_FEATURES = 1 << 16, ADAPTER_MAX_SLOTS = 1 << 16;

struct AdapterSlot {  // one entry of the device table; rank 0 = no adapter
    float scale;
    int32_t rank;
};

// Sizes of the operands in fragment order (k_adapter.hip).
struct AdapterShape {
    int32_t dtype, in, out, slots;
    int32_t kt;   // fragments along in, an even number
    int32_t nt;   // 16-row tiles along out, an even number
    int32_t rt;   // 16-row tiles along the rank (rows of A)
    int32_t rk;   // fragments along the rank (columns of B)
    int64_t a_slot, b_slot;  // elements of one adapter's A and B
};
AdapterShape adapter_shape(int32_t dtype, int32_t in, int32_t out, int32_t max_rank, int32_t slots);

// src [rows][cols] row-major to fragments [tiles][frags][64 lanes][16 bytes], zero padded; what: 0 W, 1 A, 2 B
void adapter_pack(int32_t dtype, const void* src, int rows, int cols, int tiles, int frags, int what, void* dst);
// f32 layers: W once more, as three bf16 a value in fragment order and 1 / the scale of each output
int64_t adapter_split_bytes(const AdapterShape& s);
void adapter_split(const AdapterShape& s, const float* w, void* parts, float* inv);

struct AdapterArgs {
    AdapterShape s;
    const void *w, *bias, *a, *b;  // bias nullable
    const void* w_split;           // f32: W as three bf16 a value, and 1 / the scales
    const float* w_inv;
    const AdapterSlot* slot;
    const void* x;
    const int32_t* ids;  // nullable: no adapters
    void* y;
    int64_t n;
};
void adapter_forward(const AdapterArgs& g);

}  // namespace rvx

struct rvx_adapter_linear {
    rvx::AdapterShape s;
    int32_t max_rank = 0;
    int device = 0;
    rvx::DevMem w, bias, a, b, slot, split, split_inv;
    std::vector<rvx::AdapterSlot> host_slot;
};
