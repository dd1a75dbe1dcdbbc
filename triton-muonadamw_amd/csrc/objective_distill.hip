// Distillation from a teacher's top logits for gfx950: the divergence of a row and its gradient in one pass.
#include "mamw_rows.h"

namespace mamw {
namespace {

// ---- distillation

struct Distill {
    PerRow logits, indices, lse, mask;
    int64_t items;
    int k;
    float temperature, scale;
    const int32_t* count;
};

__device__ __forceinline__ float load_float(const PerRow& a, int64_t i) {
    if (a.type == MAMW_F32) return reinterpret_cast<const float*>(a.data)[i];
    if (a.type == MAMW_BF16) return widen(reinterpret_cast<const bf16_t*>(a.data)[i]);
    return widen(reinterpret_cast<const _Float16*>(a.data)[i]);
}

// The teacher's part of a row, by one wave; the others have it after the next barrier.
struct Teacher {
    float sum_p;   // of all entries
    float x_top;   // the student's largest logit among them
    int entries;   // different ones
    int repeated;  // some are given more than once
    int beyond;    // some are outside the vocabulary
};

// An entry of LDS: its index, or kPadding, or kRepeated - its index where an entry before it has the same.
constexpr int kPadding = -1, kRepeated = -2;

// kTail: the teacher's entries are taken out of the row (an index in `marked`, a bit for each entry of the
// vocabulary) and their sum is added from the gathered logits, so that the sum over all others is not the small
// difference of two large ones.  The same bits find repeated entries; where the vocabulary is too large for them
// (bits = 0, never with kTail) every pair of entries is compared.
template <typename T, int kThreads_, int kVecs, bool kRest, bool kTail>
__global__ __launch_bounds__(kThreads_, kRowWaves<kVecs>) void distill_kernel(
    Rows x, Distill p, int bits, float4* __restrict__ partials, const float* __restrict__ scale, int unless_one,
    T* __restrict__ grad) {
    extern __shared__ uint32_t dynamic[];
    __shared__ Stats lds[kThreads_ / 64];
    __shared__ Teacher teacher;
    uint32_t* marked = dynamic;
    int32_t* index = reinterpret_cast<int32_t*>(marked + bits);
    float* logp = reinterpret_cast<float*>(index + p.k);
    float* xs = logp + p.k;
    const float f = scale ? *scale : 1.f;
    if (scale && unless_one && f == 1.f) return;
    for (int j = threadIdx.x; j < bits; j += kThreads_) marked[j] = 0;
    const int lane = threadIdx.x;
    const uint32_t r = row_of_block();
    if (r >= uint32_t(x.rows)) return;
    const Place at = place(x, r);
    T* g = grad ? grad + int64_t(r) * x.vocab : nullptr;
    if (!load_mask(p.mask, at)) {
        if (partials && threadIdx.x == 0) partials[r] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (g) zero_row(g, x.vocab, kThreads_);
        return;
    }
    const T* row = row_of<T>(x, at);
    HeldRow<T, kThreads_, kVecs, kRest> held;
    held.load(row, x.vocab);
    const float all = count_all(p.count, p.items, false);
    __syncthreads();  // the bits are clear
    if (threadIdx.x < 64) {
        const int64_t tl = offset(p.logits, at), ti = offset(p.indices, at);
        bool beyond = false, repeated = bits == 0;
#pragma unroll 1
        for (int k = lane; k < p.k; k += 64) {
            const float t = load_float(p.logits, tl + k);
            const int64_t j = load_int(p.indices, ti + k);
            const bool in = j >= 0 && j < x.vocab && t != -INFINITY;
            beyond |= j >= x.vocab;
            index[k] = in ? int32_t(j) : kPadding;
            logp[k] = t;
            xs[k] = in ? widen(row[j]) : -INFINITY;
            if (in && bits) repeated |= (atomicOr(&marked[j >> 5], 1u << (j & 31)) >> (j & 31)) & 1u;
        }
        if (__any(repeated)) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll 1
            for (int k = lane; k < p.k; k += 64) {
                int before = 0;
                const int j = index[k];
                for (int i = 0; i < k; ++i) before += index[i] == j || index[i] == kRepeated - j;
                if (j >= 0 && before) index[k] = kRepeated - j;
            }
        }
        const int any_repeated = __any(repeated), any_beyond = __any(beyond);
        if (lane == 0) {
            teacher.repeated = any_repeated;
            teacher.beyond = any_beyond;
        }
    }
    auto take_out = [&](vec_t& v, int n) {
        if constexpr (kTail) {
            // the bits of vector n: elements head + n kVec and on
            const int j = held.span.head + n * kVec<T>;
            const uint32_t w = j >> 5;
            if (n >= held.span.vecs) return;
            uint32_t m = marked[w] >> (j & 31);
            if ((j & 31) + kVec<T> > 32 && int(w) + 1 < bits) m |= marked[w + 1] << (32 - (j & 31));
            m &= (1u << kVec<T>) - 1u;
            if (m == 0) return;
            const vec_t none = nothing<T>();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (sizeof(T) == 4) {
                    if (m >> i & 1u) v[i] = none[i];
                } else {
                    const uint32_t lo = m >> (2 * i) & 1u ? 0xffffu : 0u, hi = m >> (2 * i + 1) & 1u ? 0xffff0000u : 0u;
                    v[i] = (v[i] & ~(lo | hi)) | (none[i] & (lo | hi));
                }
            }
        }
    };
    if constexpr (kTail) {
        __syncthreads();  // all bits are set
        if constexpr (!kRest)
            held.each([&](vec_t& v, int n) {
                take_out(v, n + int(threadIdx.x));
                // four vectors' bits at a time: all at once would take more registers than there are
                if (n / kThreads_ % 4 == 3) __builtin_amdgcn_sched_barrier(0);
            });
        const int j = extra_element<T>(held.span, threadIdx.x);
        if (int(threadIdx.x) < held.span.extra && (marked[j >> 5] >> (j & 31) & 1u)) held.single = -INFINITY;
    }
    if (threadIdx.x < 64) {
        float shift = 0.f, top = 0.f;
        if constexpr (kTail) {
            shift = load_f32(p.lse, at);
        } else {
            top = -INFINITY;
#pragma unroll 1
            for (int k = lane; k < p.k; k += 64) top = index[k] != kPadding ? fmaxf(top, logp[k]) : top;
            top = wave_max(top);
            float z = 0.f;
#pragma unroll 1
            for (int k = lane; k < p.k; k += 64)
                if (index[k] != kPadding) z += __builtin_amdgcn_exp2f(below(logp[k], top, x.c));
            shift = logf(wave_sum(z));
        }
        float sum_p = 0.f, x_top = -INFINITY;
        int entries = 0;
#pragma unroll 1
        for (int k = lane; k < p.k; k += 64) {
            if (index[k] == kPadding) continue;
            const float l = (logp[k] - top) * x.inv_t - shift;
            logp[k] = l;
            sum_p += expf(l);
            x_top = fmaxf(x_top, xs[k]);
            entries += index[k] >= 0;
        }
        sum_p = wave_sum(sum_p);
        x_top = wave_max(x_top);
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) entries += __shfl_xor(entries, o, 64);
        if (lane == 0) {
            teacher.sum_p = sum_p;
            teacher.x_top = x_top;
            teacher.entries = entries;
        }
    }
    const Stats wave = held.stats(x.c, take_out);
    Stats st;
    if constexpr (kTail) {
        // x_top is wave 0's: it reaches the reference through the waves' statistics
        Stats mine = wave;
        if (threadIdx.x < 64) move_to<false>(mine, fmaxf(wave.m, wave_max(lane == 0 ? teacher.x_top : -INFINITY)), x.c);
        st = over_block<false, kThreads_>(mine, x.c, lds);
    } else {
        st = over_block<false, kThreads_>(wave, x.c, lds);
    }
    const float s_out = st.s;
    if constexpr (kTail) {
        float s_in = 0.f;
#pragma unroll 1
        for (int k = threadIdx.x % 64; k < p.k; k += 64)
            if (index[k] >= 0) s_in += __builtin_amdgcn_exp2f(below(xs[k], st.m, x.c));
        st.s += wave_sum(s_in);
    }
    const bool beyond = teacher.beyond;
    float share = teacher.entries > 0 ? 1.f : 0.f;  // of q_j outside the teacher's entries
    const float in = kTail ? 1.f : share;
    float rest_loss = 0.f;
    if constexpr (kTail) {
        share = 1.f;
        if (teacher.entries < x.vocab) {
            const float rest_q = s_out / st.s, rest_p = fmaxf(1.f - teacher.sum_p, kSmallestTail);
            rest_loss = rest_p * logf(rest_p / rest_q);
            share = 1.f - rest_p / rest_q;
        }
    }
    if (threadIdx.x < 64 && partials) {
        const float log_s = logf(st.s);
        float loss = 0.f;
#pragma unroll 1
        for (int k = lane; k < p.k; k += 64) {
            if (index[k] == kPadding) continue;
            const float prob = expf(logp[k]);
            // p log p = 0 at p = 0; NaN stays
            loss += prob > 0.f ? prob * (logp[k] - ((xs[k] - st.m) * x.inv_t - log_s)) : prob;
        }
        loss = wave_sum(loss) + rest_loss;
        if (lane == 0) partials[r] = make_float4((beyond ? NAN : loss) / all, 0.f, 0.f, 0.f);
    }
    if (g) {
        const float w = beyond ? NAN : f * p.scale * p.temperature / all, inv_s = 1.f / st.s;
        held.write(g, w * share * inv_s, st.m, x.c, take_out);
        __syncthreads();  // then the entries themselves, over what was written there
        for (int k = threadIdx.x; k < p.k; k += kThreads_) {
            const int j = index[k];
            if (j < 0) continue;
            float prob = expf(logp[k]);
            if (teacher.repeated)
                for (int i = k + 1; i < p.k; ++i) prob += index[i] == kRepeated - j ? expf(logp[i]) : 0.f;
            g[j] = narrow<T>(w * (in * inv_s * __builtin_amdgcn_exp2f(below(xs[k], st.m, x.c)) - prob));
        }
    }
}

int launch_distill(const mamw_rows& x, const mamw_distill& p, const ObjectiveWorkspace& ws, float4* partials,
                   const float* scale, int unless_one, void* grad, char* base, hipStream_t stream) {
    const Rows rows = make_rows(x, p.temperature);
    if (rows.rows == 0) return MAMW_OK;
    Distill d;
    d.logits = make_per_row(p.teacher_logits);
    d.indices = make_per_row(p.teacher_indices);
    d.lse = make_per_row(p.teacher_lse);
    d.mask = make_per_row(p.mask);
    d.items = ws.items;
    d.k = int(p.k);
    d.temperature = p.temperature;
    d.scale = p.scale;
    d.count = reinterpret_cast<const int32_t*>(base);
    const bool tail = p.teacher_lse.data != nullptr;
    const int bits = x.vocab <= kMaxTailVocab ? int((x.vocab + 31) / 32) : 0;
    const size_t lds = size_t(bits) * 4 + size_t(d.k) * 12;
    return with_type(x.type, [&](auto t) {
        using T = decltype(t);
        return with_held_row(x.vocab / kVec<T>, [&](auto n, auto v, auto rest) {
            constexpr int kN = decltype(n)::value, kV = decltype(v)::value;
            constexpr bool kRest = decltype(rest)::value != 0;
            return int(launch_lds(K_OBJ_DISTILL, kN + tail, 0.0, row_bytes(x, grad != nullptr),
                                  tail ? distill_kernel<T, kN, kV, kRest, true> : distill_kernel<T, kN, kV, kRest, false>,
                                  row_grid(rows.rows), dim3(kN), lds, stream, rows, d, bits,
                                  partials, scale, unless_one, static_cast<T*>(grad)));
        });
    });
}

}  // namespace
}  // namespace mamw

using namespace mamw;

extern "C" int mamw_distill_workspace_bytes(const mamw_rows* logits, const mamw_distill* p, size_t* bytes) {
    ObjectiveWorkspace ws;
    if (!bytes) return MAMW_ERR_NULL;
    const int st = check_distill(logits, p, nullptr, &ws);
    if (st == MAMW_OK) *bytes = ws.bytes;
    return st;
}

extern "C" int mamw_distill_loss(const mamw_rows* logits, const mamw_distill* p, float* result, void* grad,
                                 void* workspace, size_t workspace_bytes, mamw_stream_t stream) {
    ObjectiveWorkspace ws;
    int st = check_distill(logits, p, grad, &ws);
    if (st != MAMW_OK) return st;
    if ((st = check_workspace(ws, workspace, workspace_bytes)) != MAMW_OK) return st;
    if (!result) return MAMW_ERR_NULL;
    const Rows rows = make_rows(*logits, p->temperature);
    char* base = static_cast<char*>(workspace);
    float4* partials = reinterpret_cast<float4*>(base + ws.partials_at);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const PerRow none = {};
    if ((st = launch_count(rows, none, 0, make_per_row(p->mask), {nullptr, 0}, ws, false, base, s)) != MAMW_OK)
        return st;
    if ((st = launch_distill(*logits, *p, ws, partials, nullptr, 0, grad, base, s)) != MAMW_OK) return st;
    return launch_result(ws, base, rows.rows, p->scale * p->temperature * p->temperature, result, s);
}

extern "C" int mamw_distill_grad(const mamw_rows* logits, const mamw_distill* p, const float* scale, int unless_one,
                                 void* grad, void* workspace, size_t workspace_bytes, mamw_stream_t stream) {
    ObjectiveWorkspace ws;
    int st = check_distill(logits, p, grad, &ws);
    if (st != MAMW_OK) return st;
    if ((st = check_workspace(ws, workspace, workspace_bytes)) != MAMW_OK) return st;
    if (!scale || (!grad && logits->outer * logits->inner > 0)) return MAMW_ERR_NULL;
    return launch_distill(*logits, *p, ws, nullptr, scale, unless_one, grad, static_cast<char*>(workspace),
                          static_cast<hipStream_t>(stream));
}
