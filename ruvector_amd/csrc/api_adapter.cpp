// api_adapter.cpp — C ABI of AdapterLinear. Arguments are checked here; the kernels assume what
// is checked.
#include <cmath>

#include "adapter.hpp"

using namespace rvx;

namespace {

void check_layer(const rvx_adapter_linear* l) {
    RVX_REQUIRE(l, RVX_ERR_INVALID_PARAMETER, "null layer");
    RVX_REQUIRE(l->device == device().id, RVX_ERR_INVALID_PARAMETER,
                "the layer is on device " + std::to_string(l->device) + ", not the current one");
}

}  // namespace

extern "C" {

rvx_status rvx_adapter_linear_create(const rvx_adapter_linear_config* cfg, const rvx_buffer* weight,
                                     const rvx_buffer* bias, rvx_adapter_linear** out) {
    return guard([&] {
        RVX_REQUIRE(cfg && out, RVX_ERR_INVALID_PARAMETER, "null argument");
        check_dtype(cfg->dtype);
        RVX_REQUIRE(cfg->in_features >= 1 && cfg->in_features <= ADAPTER_MAX_FEATURES && cfg->out_features >= 1 &&
                        cfg->out_features <= ADAPTER_MAX_FEATURES,
                    RVX_ERR_LAYER_CONFIG, "in_features and out_features must be in [1, 65536]");
        RVX_REQUIRE(cfg->max_rank >= 1 && cfg->max_rank <= ADAPTER_MAX_RANK, RVX_ERR_LAYER_CONFIG,
                    "max_rank must be in [1, 128]");
        RVX_REQUIRE(cfg->max_adapters >= 0 && cfg->max_adapters <= ADAPTER_MAX_SLOTS, RVX_ERR_LAYER_CONFIG,
                    "max_adapters must be in [0, 65536]");
        const int size = dtype_size(cfg->dtype);
        check_rows(weight, "weight", cfg->out_features, cfg->in_features, cfg->in_features, size);
        if (bias) check_rows(bias, "bias", 1, cfg->out_features, cfg->out_features, size);
        ComputeLock cl;
        auto l = std::make_unique<rvx_adapter_linear>();
        l->s = adapter_shape(cfg->dtype, cfg->in_features, cfg->out_features, cfg->max_rank, cfg->max_adapters);
        l->max_rank = cfg->max_rank;
        l->device = device().id;
        const AdapterShape& s = l->s;
        l->w.reset((int64_t)s.nt * s.kt * 1024);
        adapter_pack(s.dtype, weight->mem.p, s.out, s.in, s.nt, s.kt, 0, l->w.p);
        if (const int64_t bytes = adapter_split_bytes(s)) {
            l->split.reset(bytes);
            l->split_inv.reset((int64_t)s.out * 4);
            adapter_split(s, weight->mem.as<float>(), l->split.p, l->split_inv.as<float>());
        }
        if (bias) {
            l->bias.reset((int64_t)s.out * size);
            RVX_HIP(hipMemcpyAsync(l->bias.p, bias->mem.p, (size_t)s.out * size, hipMemcpyDeviceToDevice, stream()));
        }
        l->host_slot.assign(s.slots, AdapterSlot{0.0f, 0});
        if (s.slots) {
            l->a.reset(s.a_slot * s.slots * size);
            l->b.reset(s.b_slot * s.slots * size);
            l->slot.reset((int64_t)s.slots * sizeof(AdapterSlot));
            l->slot.upload(l->host_slot.data(), l->slot.bytes);
        }
        sync();  // the caller may free weight and bias now
        *out = l.release();
    });
}

rvx_status rvx_adapter_linear_destroy(rvx_adapter_linear* l) {
    return guard([&] { delete l; });
}

rvx_status rvx_adapter_linear_set(rvx_adapter_linear* l, int32_t slot, int32_t rank, const rvx_buffer* a,
                                  const rvx_buffer* b, float scale) {
    return guard([&] {
        check_layer(l);
        const AdapterShape& s = l->s;
        RVX_REQUIRE(slot >= 0 && slot < s.slots, RVX_ERR_INVALID_PARAMETER,
                    "slot " + std::to_string(slot) + " outside [0, " + std::to_string(s.slots) + ")");
        RVX_REQUIRE(rank >= 0 && rank <= l->max_rank, RVX_ERR_INVALID_PARAMETER,
                    "rank " + std::to_string(rank) + " outside [0, " + std::to_string(l->max_rank) + "]");
        RVX_REQUIRE(std::isfinite(scale), RVX_ERR_INVALID_PARAMETER, "scale must be finite");
        const int size = dtype_size(s.dtype);
        if (rank) {
            check_rows(a, "a", rank, s.in, s.in, size);
            check_rows(b, "b", s.out, rank, rank, size);
        }
        ComputeLock cl;
        if (rank) {
            adapter_pack(s.dtype, a->mem.p, rank, s.in, s.rt, s.kt, 1, (char*)l->a.p + slot * s.a_slot * size);
            adapter_pack(s.dtype, b->mem.p, s.out, rank, s.nt, s.rk, 2, (char*)l->b.p + slot * s.b_slot * size);
        }
        l->host_slot[slot] = AdapterSlot{scale, rank};
        l->slot.upload(&l->host_slot[slot], sizeof(AdapterSlot), (int64_t)slot * sizeof(AdapterSlot));  // waits
    });
}

rvx_status rvx_adapter_linear_forward_device(const rvx_adapter_linear* l, const rvx_buffer* x, int64_t n,
                                             const rvx_buffer* adapter_ids, rvx_buffer* y) {
    return guard([&] {
        check_layer(l);
        const AdapterShape& s = l->s;
        RVX_REQUIRE(n >= 0 && n <= ((int64_t)1 << 24), RVX_ERR_INVALID_PARAMETER, "n must be in [0, 2^24]");
        const int size = dtype_size(s.dtype);
        check_rows(x, "x", n, s.in, s.in, size);
        check_rows(y, "y", n, s.out, s.out, size);
        if (adapter_ids) check_rows(adapter_ids, "adapter_ids", n, 1, 1, 4);
        check_apart(x, y, "x and y");
        check_apart(adapter_ids, y, "adapter_ids and y");
        if (n == 0) return;
        ComputeLock cl;
        AdapterArgs g{s, l->w.p, l->bias.p, l->a.p, l->b.p, l->split.p, l->split_inv.as<float>(), l->slot.as<AdapterSlot>(), x->mem.p,
                      adapter_ids && s.slots ? adapter_ids->mem.as<int32_t>() : nullptr, y->mem.p, n};
        adapter_forward(g);
    });
}

}  // extern "C"
