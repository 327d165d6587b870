// api_heads.cpp — C ABI of the operators that train and serve the embeddings around the graph
// layers: rows of a learned table by id, and log probabilities over scores. Every argument is
// checked here, before anything is launched; the kernels assume what is checked.
#include <cmath>

#include "heads.hpp"

using namespace rvx;

namespace {

constexpr int64_t MAX_INDEX = ((int64_t)1 << 31) - 1;

void check_embedding(int32_t dtype, int64_t rows, int32_t dim, int64_t n, float scale) {
    check_dtype(dtype);
    RVX_REQUIRE(rows >= 1 && rows < MAX_INDEX, RVX_ERR_INVALID_PARAMETER, "rows must be in [1, 2^31 - 1)");
    RVX_REQUIRE(dim >= 1 && dim <= EMBED_MAX_DIM, RVX_ERR_INVALID_PARAMETER, "dim must be in [1, 65536]");
    RVX_REQUIRE(n >= 0 && n <= MAX_INDEX, RVX_ERR_INVALID_PARAMETER, "n must be in [0, 2^31)");
    RVX_REQUIRE(std::isfinite(scale), RVX_ERR_INVALID_PARAMETER, "scale must be finite");
}

void check_scores(int32_t dtype, int64_t n, int64_t c, int64_t ld, float temperature) {
    check_dtype(dtype);
    RVX_REQUIRE(n >= 0 && n <= MAX_INDEX, RVX_ERR_INVALID_PARAMETER, "n must be in [0, 2^31)");
    RVX_REQUIRE(c >= 1 && c <= MAX_INDEX, RVX_ERR_INVALID_PARAMETER, "c must be in [1, 2^31)");
    RVX_REQUIRE(ld >= c && ld <= ((int64_t)1 << 40), RVX_ERR_INVALID_PARAMETER, "a row's stride must be in [c, 2^40]");
    // (inside it the kernels' scaled differences neither overflow where they count nor vanish)
    RVX_REQUIRE(temperature >= 0x1p-100f && temperature <= 0x1p100f, RVX_ERR_INVALID_PARAMETER,
                "temperature must be in [2^-100, 2^100]");
}

float* f32_of(rvx_buffer* b) { return b ? b->mem.as<float>() : nullptr; }
const float* f32_of(const rvx_buffer* b) { return b ? b->mem.as<float>() : nullptr; }
const int64_t* i64_of(const rvx_buffer* b) { return b ? b->mem.as<int64_t>() : nullptr; }

}  // namespace

extern "C" {

rvx_status rvx_embedding_forward_device(const rvx_buffer* table, int32_t dtype, int64_t rows, int32_t dim,
                                        const rvx_buffer* ids, int64_t n, float scale, rvx_buffer* out) {
    return guard([&] {
        check_embedding(dtype, rows, dim, n, scale);
        const int size = dtype_size(dtype);
        check_rows(table, "table", rows, dim, dim, size);
        check_rows(ids, "ids", n, 1, 1, 8);
        check_rows(out, "out", n, dim, dim, size);
        check_apart(table, out, "table and out");
        check_apart(ids, out, "ids and out");
        if (n == 0) return;
        ComputeLock cl;
        embedding_forward(dtype, table->mem.p, rows, dim, i64_of(ids), n, scale, out->mem.p);
    });
}

rvx_status rvx_embedding_backward_device(const rvx_buffer* grad_out, int32_t dtype, const rvx_buffer* ids, int64_t n,
                                         int64_t rows, int32_t dim, float scale, int32_t accumulate,
                                         int32_t table_dtype, rvx_buffer* grad_table) {
    return guard([&] {
        check_embedding(dtype, rows, dim, n, scale);
        check_dtype(table_dtype);
        check_rows(grad_out, "grad_out", n, dim, dim, dtype_size(dtype));
        check_rows(ids, "ids", n, 1, 1, 8);
        check_rows(grad_table, "grad_table", rows, dim, dim, dtype_size(table_dtype));
        check_apart(grad_out, grad_table, "grad_out and grad_table");
        check_apart(ids, grad_table, "ids and grad_table");
        ComputeLock cl;
        embedding_backward(dtype, grad_out->mem.p, i64_of(ids), n, rows, dim, scale, accumulate != 0, table_dtype,
                           grad_table->mem.p);
    });
}

rvx_status rvx_log_probs_device(const rvx_buffer* scores, int32_t dtype, int64_t n, int64_t c, int64_t ld,
                                float temperature, const rvx_buffer* targets, int32_t k, rvx_buffer* logp,
                                rvx_buffer* rank, rvx_buffer* entropy, rvx_buffer* stats, rvx_buffer* top_ids,
                                rvx_buffer* top_logp) {
    return guard([&] {
        check_scores(dtype, n, c, ld, temperature);
        RVX_REQUIRE(k >= 0 && k <= LOGPROBS_MAX_K, RVX_ERR_INVALID_PARAMETER, "k must be in [0, 64]");
        RVX_REQUIRE((!logp && !rank) || targets, RVX_ERR_INVALID_PARAMETER, "logp and rank need targets");
        RVX_REQUIRE(k > 0 || (!top_ids && !top_logp), RVX_ERR_INVALID_PARAMETER, "top_ids and top_logp need k > 0");
        check_rows(scores, "scores", n, c, ld, dtype_size(dtype));
        if (targets) check_rows(targets, "targets", n, 1, 1, 8);
        struct { const rvx_buffer* b; const char* what; int64_t width; int size; } outs[] = {
            {logp, "logp", 1, 4},   {rank, "rank", 1, 8},       {entropy, "entropy", 1, 4},
            {stats, "stats", 2, 4}, {top_ids, "top_ids", k, 8}, {top_logp, "top_logp", k, 4}};
        for (int i = 0; i < 6; ++i) {
            if (!outs[i].b) continue;
            check_rows(outs[i].b, outs[i].what, n, outs[i].width, outs[i].width, outs[i].size);
            check_apart(outs[i].b, scores, "scores and an output");
            check_apart(outs[i].b, targets, "targets and an output");
            for (int j = 0; j < i; ++j) check_apart(outs[i].b, outs[j].b, "outputs");
        }
        if (n == 0 || (!logp && !rank && !entropy && !stats && !top_ids && !top_logp)) return;
        ComputeLock cl;
        const LogProbsOut out{f32_of(logp), rank ? rank->mem.as<int64_t>() : nullptr, f32_of(entropy), f32_of(stats),
                              top_ids ? top_ids->mem.as<int64_t>() : nullptr, f32_of(top_logp)};
        log_probs(dtype, scores->mem.p, n, c, ld, temperature, i64_of(targets), top_ids || top_logp ? k : 0, out);
    });
}

rvx_status rvx_log_probs_backward_device(const rvx_buffer* scores, int32_t dtype, int64_t n, int64_t c, int64_t ld,
                                         float temperature, const rvx_buffer* targets, const rvx_buffer* stats,
                                         const rvx_buffer* grad_logp, const rvx_buffer* entropy,
                                         const rvx_buffer* grad_entropy, rvx_buffer* grad, int64_t ld_grad) {
    return guard([&] {
        check_scores(dtype, n, c, ld, temperature);
        RVX_REQUIRE(ld_grad >= c && ld_grad <= ((int64_t)1 << 40), RVX_ERR_INVALID_PARAMETER,
                    "a gradient row's stride must be in [c, 2^40]");
        RVX_REQUIRE(!grad_logp || targets, RVX_ERR_INVALID_PARAMETER, "grad_logp needs targets");
        RVX_REQUIRE(!grad_entropy || entropy, RVX_ERR_INVALID_PARAMETER, "grad_entropy needs entropy");
        RVX_REQUIRE(grad != scores || ld == ld_grad, RVX_ERR_INVALID_PARAMETER,
                    "a gradient in the place of the scores needs their row stride");
        const int size = dtype_size(dtype);
        check_rows(scores, "scores", n, c, ld, size);
        check_rows(stats, "stats", n, 2, 2, 4);
        check_rows(grad, "grad", n, c, ld_grad, size);
        if (targets) check_rows(targets, "targets", n, 1, 1, 8);
        if (grad_logp) check_rows(grad_logp, "grad_logp", n, 1, 1, 4);
        if (grad_entropy) {
            check_rows(entropy, "entropy", n, 1, 1, 4);
            check_rows(grad_entropy, "grad_entropy", n, 1, 1, 4);
        }
        for (const rvx_buffer* b : {stats, targets, grad_logp, entropy, grad_entropy})
            check_apart(grad, b, "grad and an input");
        if (n == 0) return;
        ComputeLock cl;
        log_probs_backward(dtype, scores->mem.p, n, c, ld, temperature, i64_of(targets), f32_of(stats),
                           f32_of(grad_logp), f32_of(entropy), f32_of(grad_entropy), grad->mem.p, ld_grad);
    });
}

}  // extern "C"
