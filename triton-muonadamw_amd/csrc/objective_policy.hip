// The clipped policy loss for gfx950: statistics, loss and gradient of a row in one pass.
#include "mamw_rows.h"

namespace mamw {
namespace {

// ---- policy loss

struct Policy {
    PerRow tokens, old, advantages, ref;
    int64_t ignore, items;
    float low, high, kl_coef, scale;
    int by_sequence;
    const int32_t* count;
    const float* lengths;
};

// With lp the token's log-probability, ratio = exp(lp - old) and a weight w of 1 / (rows that count) or 1 / (the
// sequence's length x sequences):
//     loss  = w (-min(ratio A, clamp(ratio) A) + kl_coef (exp(d) - d - 1)),  d = ref - lp
//     slope = d loss / d lp = w (-ratio A [not clamped] + kl_coef (1 - exp(d))),  g_j = slope / T ([j = t] - q_j)
// The slope needs nothing but the row and the counts, so the row is held in registers from its one read to the write of
// its gradient.  Bound by memory: 8192 x 128256 bf16, 4843 rows that count, 1.24 GB read and 2.10 written in 586 us, 5.7
// TB/s; 4096 x 50257 fp32, 0.35 and 0.82 GB, in 207, 5.7 TB/s (a copy: 6.06).  A workgroup of the longest rows waits
// for the last of its loads most of the time (10 us of 18 a row), and no second one fits beside it.
template <typename T, int kThreads_, int kVecs, bool kRest>
__global__ __launch_bounds__(kThreads_, kRowWaves<kVecs>) void policy_kernel(
    Rows x, Policy p, float* __restrict__ logprobs, Result out, const float* __restrict__ scale,
    int unless_one, T* __restrict__ grad) {
    __shared__ Stats lds[kThreads_ / 64];
    const float f = scale ? *scale : 1.f;
    if (scale && unless_one && f == 1.f) return;
    const uint32_t r = row_of_block();
    if (r >= uint32_t(x.rows)) return;
    const Place at = place(x, r);
    const int64_t token = load_int(p.tokens, offset(p.tokens, at));
    T* g = grad ? grad + int64_t(r) * x.vocab : nullptr;
    const float length = p.by_sequence ? p.lengths[r] : 1.f;  // 0: in no sequence
    if (token == p.ignore || length == 0.f) {
        if (logprobs && threadIdx.x == 0) logprobs[r] = 0.f;
        if (g) zero_row(g, x.vocab, kThreads_);
        put_part(out, r, 0.f, 0.f, 0.f);
        return;
    }
    const T* row = row_of<T>(x, at);
    const Chosen<T> chosen(row, token, x.vocab);
    const Counts counted(p.count, p.items);
    const float old = load_f32(p.old, at), adv = load_f32(p.advantages, at);
    const float ref = p.ref.data ? load_f32(p.ref, at) : 0.f;
    HeldRow<T, kThreads_, kVecs, kRest> held;
    held.load(row, x.vocab, p.count);
    const Stats wave = over_wave<false>(held.stats(x.c, Unchanged(), Unchanged()), x.c);
    const Stats st = over_block<false, kThreads_>(wave, x.c, lds);
    const float w = 1.f / (length * counted.all());
    const float xt = chosen.value();
    const float lp = (xt - st.m) * x.inv_t - logf(st.s);
    const float ratio = expf(lp - old);
    const float bound = fminf(fmaxf(ratio, 1.f - p.low), 1.f + p.high);
    const bool clipped = bound * adv < ratio * adv;
    float loss = -(clipped ? bound : ratio) * adv, kl = 0.f;
    float slope = clipped ? 0.f : -adv * ratio;
    if (p.ref.data) {
        const float d = ref - lp, e = expm1f(d);
        kl = e - d;
        loss += p.kl_coef * kl;
        slope -= p.kl_coef * e;
    }
    if (logprobs && threadIdx.x == 0) logprobs[r] = lp;
    if (g) {
        const float a = chosen.beyond ? NAN : f * p.scale * w * slope * x.inv_t, b = -a / st.s;
        held.write(g, b, st.m, x.c, Unchanged());
        // by the thread that wrote the element: its writes stay in order
        if (!chosen.beyond && int(threadIdx.x) == owner_of<T>(held.span, int(token), kThreads_))
            g[token] = narrow<T>(a + b * __builtin_amdgcn_exp2f(below(xt, st.m, x.c)));
    }
    put_part(out, r, w * p.scale * loss, w * kl, clipped ? w : 0.f);
}

int launch_policy(const mamw_rows& x, const mamw_policy& p, const ObjectiveWorkspace& ws, float* logprobs,
                  const Result& out, const float* scale, int unless_one, void* grad, char* base, hipStream_t stream) {
    const Rows rows = make_rows(x, p.temperature);
    if (rows.rows == 0) return MAMW_OK;
    Policy d;
    d.tokens = make_per_row(p.tokens);
    d.old = make_per_row(p.old_logprobs);
    d.advantages = make_per_row(p.advantages);
    d.ref = make_per_row(p.ref_logprobs);
    d.ignore = p.ignore_index;
    d.items = ws.items;
    d.low = p.clip_low;
    d.high = p.clip_high;
    d.kl_coef = p.kl_coef;
    d.scale = p.scale;
    d.by_sequence = p.by_sequence;
    d.count = reinterpret_cast<const int32_t*>(base);
    d.lengths = reinterpret_cast<const float*>(base + ws.lengths_at);
    return with_type(x.type, [&](auto t) {
        using T = decltype(t);
        return with_held_row<false>(x.vocab / kVec<T>, [&](auto n, auto v, auto rest) {
            constexpr int kN = decltype(n)::value;
            return int(launch(K_OBJ_POLICY, kN, 0.0, row_bytes(x, grad != nullptr),
                              policy_kernel<T, kN, decltype(v)::value, decltype(rest)::value != 0>,
                              row_grid(rows.rows), dim3(kN), stream, rows, d, logprobs, out,
                              scale, unless_one, static_cast<T*>(grad)));
        });
    });
}

}  // namespace
}  // namespace mamw

using namespace mamw;

extern "C" int mamw_policy_workspace_bytes(const mamw_rows* logits, const mamw_policy* p, size_t* bytes) {
    ObjectiveWorkspace ws;
    if (!bytes) return MAMW_ERR_NULL;
    const int st = check_policy(logits, p, nullptr, &ws);
    if (st == MAMW_OK) *bytes = ws.bytes;
    return st;
}

extern "C" int mamw_policy_loss(const mamw_rows* logits, const mamw_policy* p, float* result, float* logprobs,
                                void* grad, void* workspace, size_t workspace_bytes, mamw_stream_t stream) {
    ObjectiveWorkspace ws;
    int st = check_policy(logits, p, grad, &ws);
    if (st != MAMW_OK) return st;
    if ((st = check_workspace(ws, workspace, workspace_bytes)) != MAMW_OK) return st;
    const Rows rows = make_rows(*logits, p->temperature);
    if (!result || (rows.rows > 0 && !logprobs)) return MAMW_ERR_NULL;
    char* base = static_cast<char*>(workspace);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const PerRow none = {};
    if ((st = launch_count(rows, make_per_row(p->tokens), p->ignore_index, none, {p->offsets, p->sequences}, ws,
                           p->by_sequence, base, s)) != MAMW_OK)
        return st;
    const Result out = make_result(ws, base, rows.rows, rows.rows > 0, 1.f, result);
    if ((st = launch_policy(*logits, *p, ws, logprobs, out, nullptr, 0, grad, base, s)) != MAMW_OK) return st;
    return launch_result(out, ws, base, s);
}

extern "C" int mamw_policy_grad(const mamw_rows* logits, const mamw_policy* p, const float* scale, int unless_one,
                                void* grad, void* workspace, size_t workspace_bytes, mamw_stream_t stream) {
    ObjectiveWorkspace ws;
    int st = check_policy(logits, p, grad, &ws);
    if (st != MAMW_OK) return st;
    if ((st = check_workspace(ws, workspace, workspace_bytes)) != MAMW_OK) return st;
    if (!scale || (!grad && logits->outer * logits->inner > 0)) return MAMW_ERR_NULL;
    return launch_policy(*logits, *p, ws, nullptr, Result(), scale, unless_one, grad, static_cast<char*>(workspace),
                         static_cast<hipStream_t>(stream));
}
