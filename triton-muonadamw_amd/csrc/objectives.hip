// Objectives of a training step for gfx950: token log-probabilities, policy, preference and distillation losses
// over rows of logits, with d loss / d logits.
//
// One workgroup takes one row at a time: the row's largest logit, the sum of the exponentials below it, then the
// gradient.  All of them are bound by memory: 2 or 4 bytes read a logit, as many written, and some ten operations.
#include "mamw_device.h"
#include "mamw_launch.h"
#include "mamw_objectives.h"

namespace mamw {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kSmallestTail = 0x1p-20f;

// ---- element types

struct bf16_t {
    uint16_t bits;
};

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(bf16_t x) { return bf16_to_f32(x.bits); }
__device__ __forceinline__ float widen(_Float16 x) { return float(x); }

template <typename T>
__device__ __forceinline__ T narrow(float x);  // to nearest, ties to even
template <>
__device__ __forceinline__ float narrow<float>(float x) { return x; }
template <>
__device__ __forceinline__ bf16_t narrow<bf16_t>(float x) { return {uint16_t(f32_to_bf16(x))}; }
template <>
__device__ __forceinline__ _Float16 narrow<_Float16>(float x) { return _Float16(x); }

// ---- what the kernels are given

struct Rows {
    const char* data;
    int64_t outer_stride, inner_stride;
    uint32_t inner;
    int32_t rows, vocab;
    float c, inv_t;  // log2(e) / T, 1 / T
};

struct PerRow {
    const char* data;
    int64_t outer_stride, inner_stride;
    int32_t type;
};

struct Place {
    uint32_t outer, inner;
};

__device__ __forceinline__ Place place(const Rows& x, uint32_t r) {
    const uint32_t o = r / x.inner;
    return {o, r - o * x.inner};
}

template <typename T>
__device__ __forceinline__ const T* row_of(const Rows& x, Place at) {
    return reinterpret_cast<const T*>(x.data) + (at.outer * x.outer_stride + at.inner * x.inner_stride);
}

__device__ __forceinline__ int64_t offset(const PerRow& a, Place at) {
    return at.outer * a.outer_stride + at.inner * a.inner_stride;
}
__device__ __forceinline__ float load_f32(const PerRow& a, Place at) {
    return reinterpret_cast<const float*>(a.data)[offset(a, at)];
}
__device__ __forceinline__ int64_t load_int(const PerRow& a, int64_t i) {
    return a.type == MAMW_I32 ? int64_t(reinterpret_cast<const int32_t*>(a.data)[i])
                              : reinterpret_cast<const int64_t*>(a.data)[i];
}
__device__ __forceinline__ bool load_mask(const PerRow& a, Place at) {
    return !a.data || reinterpret_cast<const uint8_t*>(a.data)[offset(a, at)] != 0;
}

// ---- reductions over the workgroup, always in the same order

template <int N>
struct Floats {
    float v[N];
};

template <int N>
__device__ __forceinline__ Floats<N> block_sum(Floats<N> x, float* lds) {
#pragma unroll
    for (int i = 0; i < N; ++i) x.v[i] = wave_sum(x.v[i]);
    const int wave = threadIdx.x / 64;
    __syncthreads();
    if (threadIdx.x % 64 == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) lds[wave * N + i] = x.v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        x.v[i] = lds[i];
        for (int w = 1; w < kWaves; ++w) x.v[i] += lds[w * N + i];
    }
    return x;
}

__device__ __forceinline__ float block_max(float x, float* lds) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) x = fmaxf(x, __shfl_xor(x, o, 64));
    __syncthreads();
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = x;
    __syncthreads();
    x = lds[0];
    for (int w = 1; w < kWaves; ++w) x = fmaxf(x, lds[w]);
    return x;
}

// ---- a row

// y_j = log2 of exp((x_j - M) / T).  The difference first: logits and masks may be the type's lowest value, whose
// product with log2(e) / T overflows.
__device__ __forceinline__ float below(float x, float m, float c) { return (x - m) * c; }

struct RowStats {
    float m, s;   // largest logit, sum of 2^y
    float sy;     // sum of 2^y y (entropies)
    float s_in;   // the part of s in marked entries
};

// `marked`: a bit for each entry, set for those that count into s_in (NULL: none).
template <typename T, bool kEntropy>
__device__ __forceinline__ RowStats row_stats(const T* __restrict__ x, const Rows& rows, const uint32_t* marked,
                                              float* lds) {
    float m = -INFINITY;
    for (int j = threadIdx.x; j < rows.vocab; j += kThreads) m = fmaxf(m, widen(x[j]));
    m = block_max(m, lds);
    Floats<3> sum = {{0.f, 0.f, 0.f}};
    for (int j = threadIdx.x; j < rows.vocab; j += kThreads) {
        const float y = below(widen(x[j]), m, rows.c);
        const float e = __builtin_amdgcn_exp2f(y);
        const bool in = marked && (marked[j >> 5] >> (j & 31) & 1u);
        sum.v[0] += in ? 0.f : e;
        sum.v[2] += in ? e : 0.f;
        // 0 * -inf: entries of no probability add nothing
        if (kEntropy) sum.v[1] += e * fmaxf(y, -1e30f);
    }
    sum = block_sum(sum, lds);
    return {m, sum.v[0] + sum.v[2], sum.v[1], sum.v[2]};
}

template <typename T>
__device__ __forceinline__ void zero_row(T* __restrict__ g, int vocab) {
    for (int j = threadIdx.x; j < vocab; j += kThreads) g[j] = narrow<T>(0.f);
}

// The logit of the row's token: NaN where it is beyond the vocabulary.
template <typename T>
__device__ __forceinline__ float chosen(const T* x, int64_t token, int vocab) {
    return token >= 0 && token < vocab ? widen(x[token]) : NAN;
}

// ---- token_logprobs

template <typename T, bool kEntropy>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(Rows x, PerRow tokens, int64_t ignore,
                                                            float* __restrict__ logprobs,
                                                            float* __restrict__ entropy, float* __restrict__ stats,
                                                            float* __restrict__ coef) {
    __shared__ float lds[kWaves * 3];
    for (uint32_t r = blockIdx.x; r < uint32_t(x.rows); r += gridDim.x) {
        const Place at = place(x, r);
        const int64_t token = load_int(tokens, offset(tokens, at));
        float lp = 0.f, h = 0.f;
        if (coef && threadIdx.x == 0) coef[r] = 0.f;  // of rows outside all sequences
        if (token != ignore) {
            const T* row = row_of<T>(x, at);
            const float xt = chosen(row, token, x.vocab);
            const RowStats st = row_stats<T, kEntropy>(row, x, nullptr, lds);
            const float log_s = logf(st.s);
            lp = (xt - st.m) * x.inv_t - log_s;
            h = log_s - kLn2 * st.sy / st.s;
            if (stats && threadIdx.x == 0) {
                stats[2 * int64_t(r)] = st.m;
                stats[2 * int64_t(r) + 1] = st.s;
            }
        }
        if (threadIdx.x == 0) {
            logprobs[r] = lp;
            if (kEntropy) entropy[r] = h;
        }
    }
}

// ---- the gradient from statistics at hand

template <typename T, bool kEntropy>
__global__ __launch_bounds__(kThreads) void logits_grad_kernel(Rows x, PerRow tokens, int64_t ignore,
                                                               const float* __restrict__ stats, PerRow coef,
                                                               PerRow entropy_coef,
                                                               const float* __restrict__ entropy,
                                                               const float* __restrict__ scale, T* __restrict__ grad) {
    const float f = (scale ? *scale : 1.f) * x.inv_t;
    for (uint32_t r = blockIdx.x; r < uint32_t(x.rows); r += gridDim.x) {
        const Place at = place(x, r);
        const int64_t token = load_int(tokens, offset(tokens, at));
        T* g = grad + int64_t(r) * x.vocab;
        if (token == ignore) {
            zero_row(g, x.vocab);
            continue;
        }
        const T* row = row_of<T>(x, at);
        const float m = stats[2 * int64_t(r)], s = stats[2 * int64_t(r) + 1], inv_s = 1.f / s;
        const bool beyond = token < 0 || token >= x.vocab;
        const float a = beyond ? NAN : f * load_f32(coef, at);
        const float h = kEntropy ? f * load_f32(entropy_coef, at) : 0.f;
        // a + h (log q + H) = b + h ln2 y
        const float b = kEntropy ? a + h * (entropy[r] - logf(s)) : a;
        for (int j = threadIdx.x; j < x.vocab; j += kThreads) {
            const float y = below(widen(row[j]), m, x.c);
            const float q = __builtin_amdgcn_exp2f(y) * inv_s;
            float d = -q * (kEntropy ? b + h * kLn2 * fmaxf(y, -1e30f) : b);
            if (j == token) d += a;
            g[j] = narrow<T>(d);
        }
    }
}

// ---- how many rows count, and of which sequence

struct Sequences {
    const int64_t* offsets;
    int64_t count;
};

// The rows of sequence i, whatever the offsets hold within the rows there are.
__device__ __forceinline__ void sequence_rows(const Sequences& s, const Rows& x, int64_t i, int64_t* from, int64_t* to) {
    if (!s.offsets) {
        *from = i * x.inner;
        *to = *from + x.inner;
        return;
    }
    const int64_t a = s.offsets[i], b = s.offsets[i + 1];
    *from = a < 0 ? 0 : a > x.rows ? x.rows : a;
    *to = b < 0 ? 0 : b > x.rows ? x.rows : b;
}

__device__ __forceinline__ bool counts(const Rows& x, const PerRow& tokens, int64_t ignore, const PerRow& mask,
                                       uint32_t r) {
    const Place at = place(x, r);
    if (tokens.data && load_int(tokens, offset(tokens, at)) == ignore) return false;
    return load_mask(mask, at);
}

// counts[i]: rows that count of sequence i, and in lengths[] for each row of the sequence; or, with no sequences
// (lengths NULL), of the kCountRows rows from i kCountRows on.
__global__ __launch_bounds__(kThreads) void count_kernel(Rows x, PerRow tokens, int64_t ignore, PerRow mask,
                                                         Sequences seqs, int32_t* __restrict__ count,
                                                         float* __restrict__ lengths) {
    __shared__ float lds[kWaves];
    int64_t from = int64_t(blockIdx.x) * kCountRows, to = min(from + kCountRows, int64_t(x.rows));
    if (lengths) sequence_rows(seqs, x, blockIdx.x, &from, &to);
    int n = 0;
    for (int64_t r = from + threadIdx.x; r < to; r += kThreads) n += counts(x, tokens, ignore, mask, uint32_t(r));
    // below 2^24 a thread; exact as floats where the sum is, too, else the weight's last bit
    const float all = block_sum(Floats<1>{{float(n)}}, lds).v[0];
    if (threadIdx.x == 0) count[blockIdx.x] = int32_t(all);
    if (lengths)
        for (int64_t r = from + threadIdx.x; r < to; r += kThreads) lengths[r] = all;
}

__global__ __launch_bounds__(kThreads) void zero_kernel(float* __restrict__ x, int64_t n) {
    const int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x;
    if (i < n) x[i] = 0.f;
}

// The number that weights are divided by: rows that count, or sequences that have any.
__device__ __forceinline__ float count_all(const int32_t* __restrict__ count, int64_t items, bool by_sequence,
                                           float* lds) {
    float n = 0.f;
    for (int64_t i = threadIdx.x; i < items; i += kThreads) n += by_sequence ? float(count[i] > 0) : float(count[i]);
    return fmaxf(block_sum(Floats<1>{{n}}, lds).v[0], 1.f);
}

// result[0..2]: the sums of the blocks' partial sums.
__global__ __launch_bounds__(kThreads) void result_kernel(const float* __restrict__ partials, int blocks, float f,
                                                          float* __restrict__ result) {
    __shared__ float lds[kWaves * 3];
    Floats<3> sum = {{0.f, 0.f, 0.f}};
    for (int i = threadIdx.x; i < blocks; i += kThreads)
#pragma unroll
        for (int k = 0; k < 3; ++k) sum.v[k] += partials[4 * i + k];
    sum = block_sum(sum, lds);
    if (threadIdx.x == 0) {
        result[0] = sum.v[0] * f;
        result[1] = sum.v[1];
        result[2] = sum.v[2];
    }
}

// ---- policy loss

struct Policy {
    PerRow tokens, old, advantages, ref;
    int64_t ignore, items;
    float low, high, kl_coef, scale;
    int by_sequence;
    const int32_t* count;
    const float* lengths;
};

template <typename T>
__global__ __launch_bounds__(kThreads) void policy_kernel(Rows x, Policy p, float* __restrict__ logprobs,
                                                          float* __restrict__ partials,
                                                          const float* __restrict__ scale, int unless_one,
                                                          T* __restrict__ grad) {
    __shared__ float lds[kWaves * 3];
    const float f = scale ? *scale : 1.f;
    if (scale && unless_one && f == 1.f) return;
    const float all = count_all(p.count, p.items, p.by_sequence, lds);
    Floats<3> sum = {{0.f, 0.f, 0.f}};
    for (uint32_t r = blockIdx.x; r < uint32_t(x.rows); r += gridDim.x) {
        const Place at = place(x, r);
        const int64_t token = load_int(p.tokens, offset(p.tokens, at));
        T* g = grad ? grad + int64_t(r) * x.vocab : nullptr;
        const float length = p.by_sequence ? p.lengths[r] : 1.f;  // 0: in no sequence
        if (token == p.ignore || length == 0.f) {
            if (logprobs && threadIdx.x == 0) logprobs[r] = 0.f;
            if (g) zero_row(g, x.vocab);
            continue;
        }
        const T* row = row_of<T>(x, at);
        const float xt = chosen(row, token, x.vocab);
        const RowStats st = row_stats<T, false>(row, x, nullptr, lds);
        const float lp = (xt - st.m) * x.inv_t - logf(st.s);
        const float ratio = expf(lp - load_f32(p.old, at)), adv = load_f32(p.advantages, at);
        const float bound = fminf(fmaxf(ratio, 1.f - p.low), 1.f + p.high);
        const bool clipped = bound * adv < ratio * adv;
        float loss = -(clipped ? bound : ratio) * adv, kl = 0.f;
        float slope = clipped ? 0.f : -adv * ratio;
        if (p.ref.data) {
            const float d = load_f32(p.ref, at) - lp, e = expm1f(d);
            kl = e - d;
            loss += p.kl_coef * kl;
            slope -= p.kl_coef * e;
        }
        const float w = 1.f / (length * all);
        sum.v[0] += w * p.scale * loss;
        sum.v[1] += w * kl;
        sum.v[2] += clipped ? w : 0.f;
        if (logprobs && threadIdx.x == 0) logprobs[r] = lp;
        if (g) {
            const float a = f * p.scale * w * slope * x.inv_t, b = a / st.s;
            for (int j = threadIdx.x; j < x.vocab; j += kThreads) {
                float d = -b * __builtin_amdgcn_exp2f(below(widen(row[j]), st.m, x.c));
                if (j == token || token < 0 || token >= x.vocab) d += a;
                g[j] = narrow<T>(d);
            }
        }
    }
    if (partials && threadIdx.x < 3) partials[4 * blockIdx.x + threadIdx.x] = sum.v[threadIdx.x];
}

// ---- preference loss

struct Preference {
    PerRow tokens;
    int64_t ignore;
    const float* ref;
    Sequences seqs;
    float beta, smoothing;
    int kind, length_average;
};

// One workgroup a pair: the sums over both sequences, the pair's loss and the rows' coefficients.
__global__ __launch_bounds__(kThreads) void pairs_kernel(Rows x, Preference p, const float* __restrict__ row_logprobs,
                                                         float* __restrict__ logprobs, float* __restrict__ rewards,
                                                         float* __restrict__ losses, float* __restrict__ coef) {
    __shared__ float lds[kWaves * 2];
    const int64_t pairs = p.seqs.count / 2, i = blockIdx.x;
    const PerRow none = {};
    int64_t from[2], to[2];
    float total[2], n[2];
    for (int k = 0; k < 2; ++k) {
        sequence_rows(p.seqs, x, i + k * pairs, &from[k], &to[k]);
        Floats<2> sum = {{0.f, 0.f}};
        for (int64_t r = from[k] + threadIdx.x; r < to[k]; r += kThreads) {
            sum.v[0] += row_logprobs[r];
            sum.v[1] += counts(x, p.tokens, p.ignore, none, uint32_t(r));
        }
        sum = block_sum(sum, lds);
        n[k] = p.length_average ? fmaxf(sum.v[1], 1.f) : 1.f;
        total[k] = sum.v[0] / n[k];
    }
    const float reward0 = p.beta * (total[0] - (p.ref ? p.ref[i] : 0.f));
    const float reward1 = p.beta * (total[1] - (p.ref ? p.ref[i + pairs] : 0.f));
    const float h = reward0 - reward1;
    float loss, slope;  // d loss / d h
    if (p.kind == MAMW_SIGMOID) {
        const float soft = log1pf(expf(-fabsf(h)));  // -log sigmoid(|h|)
        loss = (1.f - p.smoothing) * (soft + fmaxf(-h, 0.f)) + p.smoothing * (soft + fmaxf(h, 0.f));
        slope = p.smoothing - 1.f / (1.f + expf(h));
    } else if (p.kind == MAMW_IPO) {
        const float d = (h - 0.5f) / p.beta;
        loss = d * d;
        slope = 2.f * d / p.beta;
    } else {
        loss = h < 1.f ? 1.f - h : h >= 1.f ? 0.f : h;  // NaN stays
        slope = h < 1.f ? -1.f : h >= 1.f ? 0.f : h;
    }
    if (threadIdx.x == 0) {
        logprobs[i] = total[0];
        logprobs[i + pairs] = total[1];
        rewards[i] = reward0;
        rewards[i + pairs] = reward1;
        losses[i] = loss;
    }
    if (coef)
        for (int k = 0; k < 2; ++k) {
            const float c = (k ? -slope : slope) * p.beta / (float(pairs) * n[k]);
            for (int64_t r = from[k] + threadIdx.x; r < to[k]; r += kThreads) coef[r] = c;
        }
}

__global__ __launch_bounds__(kThreads) void mean_kernel(const float* __restrict__ x, int64_t n,
                                                        float* __restrict__ result) {
    __shared__ float lds[kWaves];
    float sum = 0.f;
    for (int64_t i = threadIdx.x; i < n; i += kThreads) sum += x[i];
    sum = block_sum(Floats<1>{{sum}}, lds).v[0];
    if (threadIdx.x == 0) result[0] = sum / float(n);
}

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

template <typename T, bool kTail>
__global__ __launch_bounds__(kThreads) void distill_kernel(Rows x, Distill p, float* __restrict__ partials,
                                                           const float* __restrict__ scale, int unless_one,
                                                           T* __restrict__ grad) {
    extern __shared__ uint32_t marked[];  // kTail: a bit for each entry of the vocabulary
    __shared__ float lds[kWaves * 4];
    __shared__ int32_t index[MAMW_MAX_TEACHER];
    __shared__ float logp[MAMW_MAX_TEACHER];
    __shared__ uint8_t first[MAMW_MAX_TEACHER];
    const float f = scale ? *scale : 1.f;
    if (scale && unless_one && f == 1.f) return;
    const float all = count_all(p.count, p.items, false, lds);
    float sum = 0.f;
    if (kTail)
        for (int j = threadIdx.x; j < (x.vocab + 31) / 32; j += kThreads) marked[j] = 0;
    for (uint32_t r = blockIdx.x; r < uint32_t(x.rows); r += gridDim.x) {
        const Place at = place(x, r);
        T* g = grad ? grad + int64_t(r) * x.vocab : nullptr;
        if (!load_mask(p.mask, at)) {
            if (g) zero_row(g, x.vocab);
            continue;
        }
        const T* row = row_of<T>(x, at);
        // the teacher's distribution
        const int64_t tl = offset(p.logits, at), ti = offset(p.indices, at);
        __syncthreads();
        float top = -INFINITY;
        bool beyond = false;
        for (int k = threadIdx.x; k < p.k; k += kThreads) {
            const float t = load_float(p.logits, tl + k);
            int64_t j = load_int(p.indices, ti + k);
            if (j < 0 || t == -INFINITY) j = -1;
            beyond |= j >= x.vocab;
            index[k] = int32_t(j >= x.vocab ? -1 : j);
            logp[k] = t;
            if (j >= 0) top = fmaxf(top, t);
        }
        beyond = __syncthreads_or(beyond);
        float shift;
        if (kTail) {
            shift = load_f32(p.lse, at);
        } else {
            top = block_max(top, lds);
            Floats<1> z = {{0.f}};
            for (int k = threadIdx.x; k < p.k; k += kThreads)
                if (index[k] >= 0) z.v[0] += __builtin_amdgcn_exp2f(below(logp[k], top, x.c));
            shift = logf(block_sum(z, lds).v[0]);
        }
        for (int k = threadIdx.x; k < p.k; k += kThreads) {
            logp[k] = kTail ? logp[k] * x.inv_t - shift : (logp[k] - top) * x.inv_t - shift;
            bool is_first = index[k] >= 0;
            for (int i = 0; i < k; ++i) is_first &= index[i] != index[k];
            first[k] = is_first;
            if (kTail && is_first) atomicOr(&marked[index[k] >> 5], 1u << (index[k] & 31));
        }
        __syncthreads();
        // the student's, and how far it is off
        const RowStats st = row_stats<T, false>(row, x, kTail ? marked : nullptr, lds);
        const float log_s = logf(st.s);
        Floats<3> part = {{0.f, 0.f, 0.f}};  // divergence, sum of p, entries
        for (int k = threadIdx.x; k < p.k; k += kThreads) {
            if (index[k] < 0) continue;
            const float prob = expf(logp[k]), logq = (widen(row[index[k]]) - st.m) * x.inv_t - log_s;
            part.v[0] += prob > 0.f ? prob * (logp[k] - logq) : prob;  // p log p = 0 at p = 0; NaN stays
            part.v[1] += prob;
            part.v[2] += first[k];
        }
        part = block_sum(part, lds);
        float loss = part.v[0], share = part.v[2] > 0.f ? 1.f : 0.f;  // of q_j outside the teacher's entries
        if (kTail) {
            const float rest_q = (st.s - st.s_in) / st.s;
            const float rest_p = int(part.v[2]) < x.vocab ? fmaxf(1.f - part.v[1], kSmallestTail) : 0.f;
            share = 1.f;
            if (rest_p > 0.f) {
                loss += rest_p * logf(rest_p / rest_q);
                share = 1.f - rest_p / rest_q;
            }
        }
        if (beyond) loss = share = NAN;
        sum += loss / all;
        if (g) {
            const float w = f * p.scale * p.temperature / all, inv_s = 1.f / st.s;
            const float in = kTail ? 1.f : share;
            for (int j = threadIdx.x; j < x.vocab; j += kThreads)
                g[j] = narrow<T>(w * share * inv_s * __builtin_amdgcn_exp2f(below(widen(row[j]), st.m, x.c)));
            __syncthreads();
            for (int k = threadIdx.x; k < p.k; k += kThreads) {
                if (!first[k]) continue;
                float prob = 0.f;
                for (int i = k; i < p.k; ++i) prob += index[i] == index[k] ? expf(logp[i]) : 0.f;
                const float q = inv_s * __builtin_amdgcn_exp2f(below(widen(row[index[k]]), st.m, x.c));
                g[index[k]] = narrow<T>(beyond ? NAN : w * (in * q - prob));
            }
        }
        if (kTail)
            for (int k = threadIdx.x; k < p.k; k += kThreads)
                if (index[k] >= 0) marked[index[k] >> 5] = 0;
    }
    if (partials && threadIdx.x < 3) partials[4 * blockIdx.x + threadIdx.x] = threadIdx.x ? 0.f : sum;
}

// ---- launches

Rows make_rows(const mamw_rows& x, float temperature) {
    Rows r;
    r.data = static_cast<const char*>(x.data);
    r.outer_stride = x.outer_stride;
    r.inner_stride = x.inner_stride;
    r.inner = uint32_t(x.inner);
    r.rows = int32_t(x.outer * x.inner);
    r.vocab = int32_t(x.vocab);
    r.c = kLog2e / temperature;
    r.inv_t = 1.f / temperature;
    return r;
}

PerRow make_per_row(const mamw_per_row& a) {
    return {static_cast<const char*>(a.data), a.outer_stride, a.inner_stride, a.type};
}

// fn(element type): the logits' type as a type.
template <typename Fn>
int with_type(int32_t type, Fn fn) {
    switch (type) {
        case MAMW_F32: return fn(float());
        case MAMW_BF16: return fn(bf16_t());
        default: return fn(_Float16());
    }
}

double row_bytes(const mamw_rows& x, bool grad) {
    return double(x.outer * x.inner) * double(x.vocab) * (x.type == MAMW_F32 ? 4.0 : 2.0) * (grad ? 2.0 : 1.0);
}

int launch_logprobs(const mamw_rows& x, const mamw_per_row& tokens, int64_t ignore, float temperature,
                    float* logprobs, float* entropy, float* stats, float* coef, hipStream_t stream) {
    const Rows rows = make_rows(x, temperature);
    return with_type(x.type, [&](auto t) {
        using T = decltype(t);
        return int(launch(K_OBJ_LOGPROBS, entropy ? 1 : 0, 0.0, row_bytes(x, false),
                          entropy ? logprobs_kernel<T, true> : logprobs_kernel<T, false>,
                          dim3(unsigned(row_blocks(rows.rows))), dim3(kThreads), stream, rows, make_per_row(tokens),
                          ignore, logprobs, entropy, stats, coef));
    });
}

int launch_count(const Rows& rows, const PerRow& tokens, int64_t ignore, const PerRow& mask, const Sequences& seqs,
                 const ObjectiveWorkspace& ws, bool by_sequence, char* base, hipStream_t stream) {
    if (by_sequence && seqs.offsets && rows.rows > 0) {
        const int st = int(launch(K_OBJ_COUNT, 1, 0.0, 0.0, zero_kernel, dim3(unsigned((rows.rows + kThreads - 1) / kThreads)),
                                  dim3(kThreads), stream, reinterpret_cast<float*>(base + ws.lengths_at),
                                  int64_t(rows.rows)));
        if (st != 0) return st;
    }
    if (ws.items == 0) return MAMW_OK;
    return int(launch(K_OBJ_COUNT, 0, 0.0, 0.0, count_kernel, dim3(unsigned(ws.items)), dim3(kThreads), stream, rows,
                      tokens, ignore, mask, seqs, reinterpret_cast<int32_t*>(base),
                      by_sequence ? reinterpret_cast<float*>(base + ws.lengths_at) : static_cast<float*>(nullptr)));
}

int launch_result(const ObjectiveWorkspace& ws, char* base, int blocks, float f, float* result, hipStream_t stream) {
    return int(launch(K_OBJ_RESULT, 0, 0.0, 0.0, result_kernel, dim3(1), dim3(kThreads), stream,
                      reinterpret_cast<const float*>(base + ws.partials_at), blocks, f, result));
}

int launch_policy(const mamw_rows& x, const mamw_policy& p, const ObjectiveWorkspace& ws, float* logprobs,
                  float* partials, const float* scale, int unless_one, void* grad, char* base, hipStream_t stream) {
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
        return int(launch(K_OBJ_POLICY, 0, 0.0, row_bytes(x, grad != nullptr), policy_kernel<T>,
                          dim3(unsigned(row_blocks(rows.rows))), dim3(kThreads), stream, rows, d, logprobs, partials,
                          scale, unless_one, static_cast<T*>(grad)));
    });
}

int launch_distill(const mamw_rows& x, const mamw_distill& p, const ObjectiveWorkspace& ws, float* partials,
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
    const size_t lds = tail ? size_t((x.vocab + 31) / 32) * 4 : 0;
    return with_type(x.type, [&](auto t) {
        using T = decltype(t);
        return int(launch_lds(K_OBJ_DISTILL, tail ? 1 : 0, 0.0, row_bytes(x, grad != nullptr),
                              tail ? distill_kernel<T, true> : distill_kernel<T, false>,
                              dim3(unsigned(row_blocks(rows.rows))), dim3(kThreads), lds, stream, rows, d, partials,
                              scale, unless_one, static_cast<T*>(grad)));
    });
}

}  // namespace
}  // namespace mamw

using namespace mamw;

extern "C" int mamw_token_logprobs(const mamw_rows* logits, const mamw_per_row* tokens, int64_t ignore_index,
                                   float temperature, float* logprobs, float* entropy, float* stats,
                                   mamw_stream_t stream) {
    int st = check_rows(logits, nullptr);
    if (st != MAMW_OK) return st;
    if (!tokens) return MAMW_ERR_NULL;
    const bool some = logits->outer * logits->inner > 0;
    if ((st = check_per_row(*tokens, some, MAMW_I64, MAMW_I32)) != MAMW_OK) return st;
    if ((st = check_temperature(temperature)) != MAMW_OK) return st;
    if (!some) return MAMW_OK;
    if (!logprobs) return MAMW_ERR_NULL;
    return launch_logprobs(*logits, *tokens, ignore_index, temperature, logprobs, entropy, stats,
                           nullptr, static_cast<hipStream_t>(stream));
}

extern "C" int mamw_logits_grad(const mamw_rows* logits, const mamw_per_row* tokens, int64_t ignore_index,
                                float temperature, const float* stats, const mamw_per_row* coef,
                                const mamw_per_row* entropy_coef, const float* entropy, const float* scale, void* grad,
                                mamw_stream_t stream) {
    int st = check_rows(logits, grad);
    if (st != MAMW_OK) return st;
    if (!tokens || !coef) return MAMW_ERR_NULL;
    const bool some = logits->outer * logits->inner > 0;
    if ((st = check_per_row(*tokens, some, MAMW_I64, MAMW_I32)) != MAMW_OK) return st;
    if ((st = check_per_row(*coef, some, MAMW_F32)) != MAMW_OK) return st;
    if (entropy_coef && (st = check_per_row(*entropy_coef, some, MAMW_F32)) != MAMW_OK) return st;
    if ((st = check_temperature(temperature)) != MAMW_OK) return st;
    if (!some) return MAMW_OK;
    if (!stats || !grad || (entropy_coef && !entropy)) return MAMW_ERR_NULL;
    const Rows rows = make_rows(*logits, temperature);
    const PerRow none = {};
    return with_type(logits->type, [&](auto t) {
        using T = decltype(t);
        return int(launch(K_OBJ_GRAD, entropy_coef ? 1 : 0, 0.0, row_bytes(*logits, true),
                          entropy_coef ? logits_grad_kernel<T, true> : logits_grad_kernel<T, false>,
                          dim3(unsigned(row_blocks(rows.rows))), dim3(kThreads), static_cast<hipStream_t>(stream),
                          rows, make_per_row(*tokens), ignore_index, stats, make_per_row(*coef),
                          entropy_coef ? make_per_row(*entropy_coef) : none, entropy, scale, static_cast<T*>(grad)));
    });
}

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
    float* partials = reinterpret_cast<float*>(base + ws.partials_at);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const PerRow none = {};
    if ((st = launch_count(rows, make_per_row(p->tokens), p->ignore_index, none, {p->offsets, p->sequences}, ws,
                           p->by_sequence, base, s)) != MAMW_OK)
        return st;
    if ((st = launch_policy(*logits, *p, ws, logprobs, partials, nullptr, 0, grad, base, s)) != MAMW_OK) return st;
    return launch_result(ws, base, row_blocks(rows.rows), 1.f, result, s);
}

extern "C" int mamw_policy_grad(const mamw_rows* logits, const mamw_policy* p, const float* scale, int unless_one,
                                void* grad, void* workspace, size_t workspace_bytes, mamw_stream_t stream) {
    ObjectiveWorkspace ws;
    int st = check_policy(logits, p, grad, &ws);
    if (st != MAMW_OK) return st;
    if ((st = check_workspace(ws, workspace, workspace_bytes)) != MAMW_OK) return st;
    if (!scale || (!grad && logits->outer * logits->inner > 0)) return MAMW_ERR_NULL;
    return launch_policy(*logits, *p, ws, nullptr, nullptr, scale, unless_one, grad, static_cast<char*>(workspace),
                         static_cast<hipStream_t>(stream));
}

extern "C" int mamw_preference_workspace_bytes(const mamw_rows* logits, const mamw_preference* p, size_t* bytes) {
    ObjectiveWorkspace ws;
    if (!bytes) return MAMW_ERR_NULL;
    const int st = check_preference(logits, p, &ws);
    if (st == MAMW_OK) *bytes = ws.bytes;
    return st;
}

extern "C" int mamw_preference_loss(const mamw_rows* logits, const mamw_preference* p, float* result, float* logprobs,
                                    float* rewards, float* stats, float* coef, void* workspace,
                                    size_t workspace_bytes, mamw_stream_t stream) {
    ObjectiveWorkspace ws;
    int st = check_preference(logits, p, &ws);
    if (st != MAMW_OK) return st;
    if ((st = check_workspace(ws, workspace, workspace_bytes)) != MAMW_OK) return st;
    if (!result || !logprobs || !rewards) return MAMW_ERR_NULL;
    const Rows rows = make_rows(*logits, p->temperature);
    char* base = static_cast<char*>(workspace);
    float* row_logprobs = reinterpret_cast<float*>(base + ws.lengths_at);
    float* losses = reinterpret_cast<float*>(base + ws.partials_at);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (rows.rows > 0 && (st = launch_logprobs(*logits, p->tokens, p->ignore_index, p->temperature, row_logprobs,
                                               nullptr, stats, coef, s)) != MAMW_OK)
        return st;
    Preference d;
    d.tokens = make_per_row(p->tokens);
    d.ignore = p->ignore_index;
    d.ref = p->ref_logprobs;
    d.seqs = {p->offsets, p->sequences};
    d.beta = p->beta;
    d.smoothing = p->smoothing;
    d.kind = p->kind;
    d.length_average = p->length_average;
    if ((st = int(launch(K_OBJ_PAIRS, 0, 0.0, 0.0, pairs_kernel, dim3(unsigned(p->sequences / 2)), dim3(kThreads), s,
                         rows, d, static_cast<const float*>(row_logprobs), logprobs, rewards, losses, coef))) != 0)
        return st;
    return int(launch(K_OBJ_RESULT, 1, 0.0, 0.0, mean_kernel, dim3(1), dim3(kThreads), s,
                      static_cast<const float*>(losses), p->sequences / 2, result));
}

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
    float* partials = reinterpret_cast<float*>(base + ws.partials_at);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const PerRow none = {};
    if ((st = launch_count(rows, none, 0, make_per_row(p->mask), {nullptr, 0}, ws, false, base, s)) != MAMW_OK)
        return st;
    if ((st = launch_distill(*logits, *p, ws, partials, nullptr, 0, grad, base, s)) != MAMW_OK) return st;
    return launch_result(ws, base, row_blocks(rows.rows), p->scale * p->temperature * p->temperature, result, s);
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
