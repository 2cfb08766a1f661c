// C ABI of the operators between sparse rows and dense matrices: argument checks and launches.  Nothing here allocates or
// waits, and no exception is thrown.
#include "dense_rows.h"

using namespace sdrb;

namespace {

constexpr uint64_t kMaxCols = 1ull << 24, kMaxRows = 0x7FFFFFFEull;

int refuse(int code, const char* what, const char* why) {
    set_error("%s: %s", what, why);
    return code;
}

int check_rows(const char* what, const sdrb_rows* rows) {
    if (!rows) return refuse(SDRB_ERR_INVALID_ARG, what, "rows is null");
    if (rows->id_bits != 32 && rows->id_bits != 64) return refuse(SDRB_ERR_INVALID_ARG, what, "id_bits must be 32 or 64");
    if (rows->n_rows > kMaxRows || rows->n_elems > 0xFFFFFFFFull)
        return refuse(SDRB_ERR_OVERFLOW, what, "more than 2^31-2 rows or 2^32-1 elements in one call");
    if (rows->n_elems && !rows->ids) return refuse(SDRB_ERR_INVALID_ARG, what, "ids is null");
    if (!rows->row_offsets && (rows->n_rows ? rows->n_elems % rows->n_rows != 0 : rows->n_elems != 0))
        return refuse(SDRB_ERR_INVALID_ARG, what, "without row_offsets n_elems must be a multiple of n_rows");
    return SDRB_OK;
}

int check_dense(const char* what, const char* name, const sdrb_dense* m) {
    const char* why = !m                                                               ? "is null"
                      : m->type != SDRB_F32 && m->type != SDRB_F16 && m->type != SDRB_BF16 ? "has an unknown type"
                      : m->n_rows && m->n_cols && !m->data                             ? "has no data"
                      : m->ld < m->n_cols                                              ? "has ld < n_cols"
                                                                                       : nullptr;
    if (why) {
        set_error("%s: %s %s", what, name, why);
        return SDRB_ERR_INVALID_ARG;
    }
    if (m->n_cols > kMaxCols || m->n_rows > kMaxRows || m->ld > (1ull << 40)) {
        set_error("%s: %s has more than 2^24 columns, 2^31-2 rows or 2^40 elements a row", what, name);
        return SDRB_ERR_OVERFLOW;
    }
    if (reinterpret_cast<uintptr_t>(m->data) % type_size(m->type) != 0) {
        set_error("%s: %s is not aligned to its elements", what, name);
        return SDRB_ERR_INVALID_ARG;
    }
    return SDRB_OK;
}

// An output over an input: rows are written while others are read.  (Matrices side by side in one buffer share its addresses, not
// their first element.)
int check_apart(const char* what, const char* name, const sdrb_dense* in, const sdrb_dense* out) {
    if (in->data != out->data || in->n_rows * in->n_cols == 0 || out->n_rows * out->n_cols == 0) return SDRB_OK;
    set_error("%s: out is %s itself", what, name);
    return SDRB_ERR_INVALID_ARG;
}

int check_scratch(const char* what, size_t need, const void* scratch, size_t bytes) {
    if (need && (!scratch || bytes < need)) {
        set_error("%s: needs %zu bytes of scratch, got %zu", what, need, scratch ? bytes : (size_t)0);
        return SDRB_ERR_INVALID_ARG;
    }
    if (need && reinterpret_cast<uintptr_t>(scratch) % 16 != 0) return refuse(SDRB_ERR_INVALID_ARG, what, "scratch is not 16-byte aligned");
    return SDRB_OK;
}

int check_spec(const char* what, const sdrb_winners_spec* w, uint64_t n_ids) {
    if (!w) return refuse(SDRB_ERR_INVALID_ARG, what, "spec is null");
    if (w->score != SDRB_SCORE_SOFTMAX && w->score != SDRB_SCORE_SIGMOID) return refuse(SDRB_ERR_INVALID_ARG, what, "unknown score");
    if (n_ids > kWinnersMaxIds || w->k > kWinnersMaxK || w->groups > kWinnersMaxGroups)
        return refuse(SDRB_ERR_UNSUPPORTED, what, "takes at most 16384 ids, k of 1024 and 256 groups");
    if (w->k < 1 || w->k > n_ids) return refuse(SDRB_ERR_INVALID_ARG, what, "k must be 1 .. ids");
    if (w->groups < 1 || n_ids % w->groups != 0 || w->top_groups < 1 || w->top_groups > w->groups || w->group_top < 1 || w->group_top > 2)
        return refuse(SDRB_ERR_INVALID_ARG, what, "groups must divide the ids, top_groups be 1 .. groups and group_top 1 or 2");
    return SDRB_OK;
}

int no_device(int device) {
    set_error("hipSetDevice(%d) failed", device);
    return SDRB_ERR_HIP;
}

}  // namespace

extern "C" {

int sdrb_batch_rows(const sdrb_batch* batch, sdrb_rows* rows) {
    if (!batch || !rows || !batch->d_offsets) return refuse(SDRB_ERR_INVALID_ARG, "sdrb_batch_rows", "null argument or no uploaded rows");
    rows->n_rows = batch->n_rows;
    rows->n_elems = batch->nnz;
    rows->row_offsets = batch->d_offsets;
    rows->ids = batch->d_ids;
    rows->weights = has_payload(batch) ? batch->d_data : nullptr;
    rows->id_bits = batch->id_bits;
    return SDRB_OK;
}

int sdrb_lookup_scratch(const sdrb_rows* rows, uint64_t n_cols, size_t* bytes) {
    const char* what = "sdrb_lookup_scratch";
    if (const int rc = check_rows(what, rows)) return rc;
    if (!bytes || n_cols > kMaxCols) return refuse(SDRB_ERR_INVALID_ARG, what, "bytes is null or n_cols above 2^24");
    *bytes = partial_bytes(segment_chunk(rows->n_rows, rows->n_elems, (uint32_t)n_cols, rows->row_offsets != nullptr), rows->n_elems, (uint32_t)n_cols);
    return SDRB_OK;
}

int sdrb_lookup(int device, const sdrb_rows* rows, const sdrb_dense* table, float scale, const sdrb_dense* out, void* scratch,
                size_t scratch_bytes, void* stream) {
    const char* what = "sdrb_lookup";
    TraceRange range(what);
    if (const int rc = check_rows(what, rows)) return rc;
    if (const int rc = check_dense(what, "table", table)) return rc;
    if (const int rc = check_dense(what, "out", out)) return rc;
    if (out->n_rows != rows->n_rows || out->n_cols != table->n_cols)
        return refuse(SDRB_ERR_INVALID_ARG, what, "out must have a row for every row and the table's columns");
    if (const int rc = check_apart(what, "table", table, out)) return rc;
    if (out->n_rows == 0 || out->n_cols == 0) return SDRB_OK;
    const uint32_t chunk = segment_chunk(rows->n_rows, rows->n_elems, (uint32_t)out->n_cols, rows->row_offsets != nullptr);
    const size_t need = partial_bytes(chunk, rows->n_elems, (uint32_t)out->n_cols);
    if (const int rc = check_scratch(what, need, scratch, scratch_bytes)) return rc;
    DeviceGuard guard(device);
    if (!guard.ok) return no_device(device);
    GatherSum g{};
    g.n_segments = rows->n_rows;
    g.n_elems = rows->n_elems;
    g.start = rows->row_offsets;
    g.index = rows->ids;
    g.index_bits = rows->id_bits;
    g.weight = rows->weights;
    g.src = table->data;
    g.src_type = table->type;
    g.src_rows = table->n_rows;
    g.src_ld = table->ld;
    g.dim = (uint32_t)out->n_cols;
    g.out = out->data;
    g.out_type = out->type;
    g.out_ld = out->ld;
    g.scale = scale;
    g.chunk = chunk;
    g.partials = static_cast<float*>(scratch);
    return launch_gather_sum(g, static_cast<hipStream_t>(stream));
}

int sdrb_lookup_grad_table_scratch(const sdrb_rows* rows, uint64_t n_table_rows, uint64_t n_cols, size_t* bytes) {
    const char* what = "sdrb_lookup_grad_table_scratch";
    if (const int rc = check_rows(what, rows)) return rc;
    if (!bytes || n_cols > kMaxCols || n_table_rows > kMaxRows)
        return refuse(SDRB_ERR_INVALID_ARG, what, "bytes is null, n_cols above 2^24 or n_table_rows above 2^31-2");
    *bytes = table_grad_scratch_bytes(*rows, n_table_rows, (uint32_t)n_cols);
    return SDRB_OK;
}

int sdrb_lookup_grad_table(int device, const sdrb_rows* rows, const sdrb_dense* grad, float scale, int accumulate,
                           const sdrb_dense* out, void* scratch, size_t scratch_bytes, void* stream) {
    const char* what = "sdrb_lookup_grad_table";
    TraceRange range(what);
    if (const int rc = check_rows(what, rows)) return rc;
    if (const int rc = check_dense(what, "grad", grad)) return rc;
    if (const int rc = check_dense(what, "out", out)) return rc;
    if (grad->n_rows != rows->n_rows || grad->n_cols != out->n_cols)
        return refuse(SDRB_ERR_INVALID_ARG, what, "grad must have a row for every row and the columns of out");
    if (const int rc = check_apart(what, "grad", grad, out)) return rc;
    if (out->n_rows == 0 || out->n_cols == 0) return SDRB_OK;
    const size_t need = table_grad_scratch_bytes(*rows, out->n_rows, (uint32_t)out->n_cols);
    if (const int rc = check_scratch(what, need, scratch, scratch_bytes)) return rc;
    DeviceGuard guard(device);
    if (!guard.ok) return no_device(device);
    return launch_table_grad(*rows, *grad, scale, accumulate != 0, *out, scratch, static_cast<hipStream_t>(stream));
}

int sdrb_lookup_grad_weights(int device, const sdrb_rows* rows, const sdrb_dense* grad, const sdrb_dense* table, float scale,
                             float* out, void* stream) {
    const char* what = "sdrb_lookup_grad_weights";
    TraceRange range(what);
    if (const int rc = check_rows(what, rows)) return rc;
    if (const int rc = check_dense(what, "grad", grad)) return rc;
    if (const int rc = check_dense(what, "table", table)) return rc;
    if (grad->n_rows != rows->n_rows || grad->n_cols != table->n_cols)
        return refuse(SDRB_ERR_INVALID_ARG, what, "grad must have a row for every row and the table's columns");
    if (rows->n_elems == 0) return SDRB_OK;
    if (!out) return refuse(SDRB_ERR_INVALID_ARG, what, "out is null");
    DeviceGuard guard(device);
    if (!guard.ok) return no_device(device);
    return launch_weight_grad(*rows, *grad, *table, scale, out, static_cast<hipStream_t>(stream));
}

int sdrb_winners(int device, const sdrb_dense* scores, const sdrb_winners_spec* spec, int32_t* out_ids, float* out_weights,
                 void* stream) {
    const char* what = "sdrb_winners";
    TraceRange range(what);
    if (const int rc = check_dense(what, "scores", scores)) return rc;
    if (const int rc = check_spec(what, spec, scores->n_cols)) return rc;
    if (scores->n_rows == 0) return SDRB_OK;
    if (!out_ids || !out_weights) return refuse(SDRB_ERR_INVALID_ARG, what, "an output is null");
    DeviceGuard guard(device);
    if (!guard.ok) return no_device(device);
    return launch_winners(*scores, *spec, out_ids, out_weights, static_cast<hipStream_t>(stream));
}

int sdrb_winners_grad(int device, const sdrb_dense* scores, const sdrb_winners_spec* spec, const int32_t* ids,
                      const float* grad_weights, const sdrb_dense* out, void* stream) {
    const char* what = "sdrb_winners_grad";
    TraceRange range(what);
    if (const int rc = check_dense(what, "scores", scores)) return rc;
    if (const int rc = check_dense(what, "out", out)) return rc;
    if (const int rc = check_spec(what, spec, scores->n_cols)) return rc;
    if (out->n_rows != scores->n_rows || out->n_cols != scores->n_cols)
        return refuse(SDRB_ERR_INVALID_ARG, what, "out must have the shape of the scores");
    if (const int rc = check_apart(what, "scores", scores, out)) return rc;
    if (scores->n_rows == 0) return SDRB_OK;
    if (!ids || !grad_weights) return refuse(SDRB_ERR_INVALID_ARG, what, "ids or grad_weights is null");
    DeviceGuard guard(device);
    if (!guard.ok) return no_device(device);
    return launch_winners_grad(*scores, *spec, ids, grad_weights, *out, static_cast<hipStream_t>(stream));
}

}  // extern "C"
