// Host-side validation of the objectives' entry points (no HIP calls).
#include "mamw_objectives.h"

#include <math.h>

#include "mamw_plan.h"

namespace mamw {

namespace {

size_t element_size(int32_t type) {
    switch (type) {
        case MAMW_F32: case MAMW_I32: return 4;
        case MAMW_BF16: case MAMW_F16: return 2;
        case MAMW_I64: return 8;
        case MAMW_BOOL: return 1;
        default: return 0;
    }
}

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

size_t round_up(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace

ObjectiveWorkspace objective_workspace(int64_t items, int64_t lengths, int64_t partials) {
    ObjectiveWorkspace w;
    w.items = items;
    w.ticket_at = round_up(size_t(items) * 4);
    w.lengths_at = w.ticket_at + 256 + round_up(kResultBlocks * 16);
    w.partials_at = w.lengths_at + round_up(size_t(lengths) * 4);
    w.bytes = w.partials_at + round_up(size_t(partials) * 4);
    return w;
}

int check_rows(const mamw_rows* x, const void* grad) {
    if (!x) return MAMW_ERR_NULL;
    if (x->type != MAMW_F32 && x->type != MAMW_BF16 && x->type != MAMW_F16) return MAMW_ERR_HYPER;
    if (x->reserved) return MAMW_ERR_HYPER;
    if (x->outer < 0 || x->inner < 0 || x->vocab < 1 || x->vocab > int64_t(1) << 30) return MAMW_ERR_SHAPE;
    if (x->outer_stride < 0 || x->inner_stride < 0) return MAMW_ERR_SHAPE;
    const int64_t most = int64_t(0x7fffffff);
    if (x->outer > most || x->inner > most || x->outer * x->inner > most) return MAMW_ERR_COUNT;
    if (x->outer * x->inner == 0) return MAMW_OK;
    if (!x->data) return MAMW_ERR_NULL;
    const size_t size = element_size(x->type);
    // Offsets are formed in 64-bit bytes on the device.
    const double last = double(x->outer - 1) * double(x->outer_stride) + double(x->inner - 1) * double(x->inner_stride) +
                        double(x->vocab);
    if (last * double(size) > 4e18 || double(x->outer * x->inner) * double(x->vocab) * double(size) > 4e18)
        return MAMW_ERR_NUMEL;
    if (!aligned(x->data, size) || !aligned(grad, size)) return MAMW_ERR_ALIGN;
    if (grad) {
        const size_t span = size_t((x->outer - 1) * x->outer_stride + (x->inner - 1) * x->inner_stride + x->vocab) * size;
        if (ranges_overlap(x->data, span, grad, size_t(x->outer * x->inner) * size_t(x->vocab) * size))
            return MAMW_ERR_ALIAS;
    }
    return MAMW_OK;
}

int check_per_row(const mamw_per_row& a, bool needed, int32_t type, int32_t other_type) {
    if (!a.data) return needed ? MAMW_ERR_NULL : MAMW_OK;
    const size_t size = element_size(a.type);  // 0: no type, whatever the caller's is compared with
    if (a.reserved || size == 0 || (a.type != type && a.type != other_type)) return MAMW_ERR_HYPER;
    if (a.outer_stride < 0 || a.inner_stride < 0) return MAMW_ERR_SHAPE;
    if (!aligned(a.data, size)) return MAMW_ERR_ALIGN;
    return MAMW_OK;
}

int check_temperature(float t) {
    // log2(e) / t has to be a number, and not nothing.
    const float c = 1.44269504f / t;
    return t > 0.f && isfinite(t) && isfinite(c) && c >= 1.17549435e-38f ? MAMW_OK : MAMW_ERR_HYPER;
}

namespace {

int check_sequences(const mamw_rows* x, const int64_t* offsets, int64_t sequences) {
    if (sequences < 0 || sequences > int64_t(0x7fffffff)) return MAMW_ERR_COUNT;
    if (!offsets && sequences != x->outer) return MAMW_ERR_COUNT;
    if (offsets && !aligned(offsets, 8)) return MAMW_ERR_ALIGN;
    return MAMW_OK;
}

int64_t count_items(int64_t rows) { return (rows + kCountRows - 1) / kCountRows; }

}  // namespace

int check_policy(const mamw_rows* x, const mamw_policy* p, const void* grad, ObjectiveWorkspace* ws) {
    if (!p) return MAMW_ERR_NULL;
    int st = check_rows(x, grad);
    if (st != MAMW_OK) return st;
    const int64_t rows = x->outer * x->inner;
    const bool some = rows > 0;
    if ((st = check_per_row(p->tokens, some, MAMW_I64, MAMW_I32)) != MAMW_OK) return st;
    if ((st = check_per_row(p->old_logprobs, some, MAMW_F32)) != MAMW_OK) return st;
    if ((st = check_per_row(p->advantages, some, MAMW_F32)) != MAMW_OK) return st;
    if ((st = check_per_row(p->ref_logprobs, false, MAMW_F32)) != MAMW_OK) return st;
    if ((st = check_sequences(x, p->offsets, p->sequences)) != MAMW_OK) return st;
    if ((st = check_temperature(p->temperature)) != MAMW_OK) return st;
    if (!(p->clip_low >= 0.f) || !(p->clip_high >= 0.f) || !isfinite(p->kl_coef) || !isfinite(p->scale))
        return MAMW_ERR_HYPER;
    *ws = p->by_sequence ? objective_workspace(p->sequences < kCountGroups ? p->sequences : kCountGroups, rows, 4 * rows)
                         : objective_workspace(count_items(rows), 0, 4 * rows);
    return MAMW_OK;
}

int check_preference(const mamw_rows* x, const mamw_preference* p, ObjectiveWorkspace* ws) {
    if (!p) return MAMW_ERR_NULL;
    int st = check_rows(x, nullptr);
    if (st != MAMW_OK) return st;
    const int64_t rows = x->outer * x->inner;
    if ((st = check_per_row(p->tokens, rows > 0, MAMW_I64, MAMW_I32)) != MAMW_OK) return st;
    if (!aligned(p->ref_logprobs, 4)) return MAMW_ERR_ALIGN;
    if (p->sequences < 2 || p->sequences % 2) return MAMW_ERR_COUNT;
    if ((st = check_sequences(x, p->offsets, p->sequences)) != MAMW_OK) return st;
    if ((st = check_temperature(p->temperature)) != MAMW_OK) return st;
    if (!(p->beta > 0.f) || !isfinite(p->beta) || !(p->smoothing >= 0.f) || !(p->smoothing <= 1.f))
        return MAMW_ERR_HYPER;
    if (p->kind < MAMW_SIGMOID || p->kind > MAMW_HINGE || p->reserved) return MAMW_ERR_HYPER;
    if (p->kind != MAMW_SIGMOID && p->smoothing != 0.f) return MAMW_ERR_HYPER;
    // The rows' log-probabilities, and one loss a pair.
    *ws = objective_workspace(0, rows, 2 * p->sequences);
    return MAMW_OK;
}

int check_distill(const mamw_rows* x, const mamw_distill* p, const void* grad, ObjectiveWorkspace* ws) {
    if (!p) return MAMW_ERR_NULL;
    int st = check_rows(x, grad);
    if (st != MAMW_OK) return st;
    const int64_t rows = x->outer * x->inner;
    const bool some = rows > 0;
    const int32_t t = p->teacher_logits.type;
    if (p->k < 1 || p->k > MAMW_MAX_TEACHER) return MAMW_ERR_SHAPE;
    if ((st = check_per_row(p->teacher_logits, some, t == MAMW_BF16 || t == MAMW_F16 ? t : MAMW_F32)) != MAMW_OK)
        return st;
    if ((st = check_per_row(p->teacher_indices, some, MAMW_I64, MAMW_I32)) != MAMW_OK) return st;
    if ((st = check_per_row(p->teacher_lse, false, MAMW_F32)) != MAMW_OK) return st;
    if ((st = check_per_row(p->mask, false, MAMW_BOOL)) != MAMW_OK) return st;
    if ((st = check_temperature(p->temperature)) != MAMW_OK) return st;
    if (!isfinite(p->scale)) return MAMW_ERR_HYPER;
    if (p->teacher_lse.data && x->vocab > kMaxTailVocab) return MAMW_ERR_SHAPE;
    // Each row's entries (index, probability), its part of the result and what there is to know of its teacher.
    *ws = objective_workspace(count_items(rows), 2 * rows * p->k, 8 * rows);
    return MAMW_OK;
}

int check_workspace(const ObjectiveWorkspace& ws, const void* workspace, size_t bytes) {
    return workspace && aligned(workspace, 256) && bytes >= ws.bytes ? MAMW_OK : MAMW_ERR_WORKSPACE;
}

}  // namespace mamw
