// Objectives of a training step for gfx950: token log-probabilities, policy, preference and distillation losses
// over rows of logits, with d loss / d logits.  Here the log-probabilities, the gradient from statistics at hand, the
// preference loss and what all have in common; objective_policy.hip and objective_distill.hip hold the others.
//
// All are bound by memory: 2 or 4 bytes read a logit, as many written, and some ten operations.  One workgroup takes
// a row.  Where the gradient of a row needs nothing beyond it (policy, distillation), the row stays in registers
// between its one read and the write of its gradient; where it does (the loss of a pair, a gradient from outside),
// a first kernel leaves the row's largest logit and sum and a second one reads the logits again.
#include "mamw_rows.h"

namespace mamw {
namespace {

// ---- token_logprobs

// log q_t = (x_t - m) / T - log s and H = log s - sum 2^y y ln2 / s, with m the largest logit and s the sum of
// exp((x - m) / T), both kept as the row goes by: a thread moves its sums when its largest logit grows, so that one read
// is enough.  Bound by that read and, nearly as much, by eleven operations an element with entropies (VALU busy 0.9 of
// the time): 5417 of 8192 rows of 50257 bf16 that count, 545 MB, in 83 us, 6.5 TB/s (a kernel that only reads: 7.0); the
// statistics of 5101 of 6000, without entropies, in 87.
template <typename T, int kThreads_, bool kEntropy>
__global__ __launch_bounds__(kThreads_) void logprobs_kernel(Rows x, PerRow tokens, int64_t ignore,
                                                             float* __restrict__ logprobs,
                                                             float* __restrict__ entropy, float* __restrict__ stats,
                                                             float* __restrict__ coef,
                                                             uint32_t* __restrict__ ticket, uint32_t keep_from) {
    __shared__ Stats lds[2][kThreads_ / 64];
    const uint32_t r = row_of_block();
    if (r >= uint32_t(x.rows)) return;
    const Place at = place(x, r);
    const int64_t token = load_int(tokens, offset(tokens, at));
    float lp = 0.f, h = 0.f;
    if (coef && threadIdx.x == 0) coef[r] = 0.f;  // of rows outside all sequences
    if (ticket && r == 0 && threadIdx.x == 0) *ticket = 0;
    if (token != ignore) {
        const T* row = row_of<T>(x, at);
        const Chosen<T> chosen(row, token, x.vocab);
        const Span span = span_of(row, x.vocab);
        auto stats_of_row = [&](auto quick) {
            constexpr bool kQuick = decltype(quick)::value != 0;
            Stats st = no_stats();
            for (int e = threadIdx.x; e < span.extra; e += kThreads_) {
                const float single = widen(row[extra_element<T>(span, e)]);
                move_to<kEntropy>(st, fmaxf(st.m, single), x.c);
                add<kEntropy>(st, single, reference(st.m), x.c);
            }
            if (kQuick && r >= keep_from)
                read_vecs<T, kEntropy, kQuick, kThreads_, true>(st, row + span.head, 0, span.vecs, x.c, Unchanged());
            else
                read_vecs<T, kEntropy, kQuick, kThreads_>(st, row + span.head, 0, span.vecs, x.c, Unchanged());
            return over_block<kEntropy, kThreads_>(over_wave<kEntropy>(st, x.c), x.c, lds[!kQuick]);
        };
        Stats st = stats_of_row(Int<1>());
        if (!quick_holds<kEntropy>(st, x.c)) st = stats_of_row(Int<0>());
        const float log_s = logf(st.s);
        lp = (chosen.value() - st.m) * x.inv_t - log_s;
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

// ---- the gradient from statistics at hand

// A workgroup takes kGradVecs vectors of one row: it waits for nothing, so short-lived ones in great number come
// nearest to a copy (6000 x 50257 bf16: 224 us with eight vectors a thread, 209 with four, 198 with two, 204 with
// one).  Rows are taken from the last: those the statistics were taken of last are still in the memory-side cache of 256
// MB (198 -> 183 us; 176 with rows from the 128-byte boundary on).
//
// g_j = (c / T) ([j = t] - q_j) - (h / T) q_j (log q_j + H), with c and h the factors of the row's log-probability and
// entropy.  Bound by memory: 513 MB read and 603 written in 176 us, 6.3 TB/s; 4096 x 128256 bf16, 630 and 1051 MB, in
// 276, 6.1 TB/s (a copy: 6.06).
constexpr int kGradUnroll = 2;
constexpr int kGradVecs = kThreads * kGradUnroll;
// Logits that the statistics leave there, rows that do not count among them.  More than it holds where many do not: with
// 400, 250, 200 and 0 MB, both directions of 6000 x 50257 bf16 take 268, 269, 268 and 269 us and of 4096 x 128256 380,
// 387, 391 and 394, with six rows of ten that count.  Where every row does it gains nothing: 296, 296, 296 and 290 us,
// and 510, 514, 513 and 510.
constexpr double kKeptBytes = 400e6;

template <typename T, bool kEntropy>
__global__ __launch_bounds__(kThreads) void logits_grad_kernel(Rows x, PerRow tokens, int64_t ignore,
                                                               const float* __restrict__ stats, PerRow coef,
                                                               PerRow entropy_coef,
                                                               const float* __restrict__ entropy,
                                                               const float* __restrict__ scale,
                                                               T* __restrict__ grad) {
    const float f = (scale ? *scale : 1.f) * x.inv_t;
    const uint32_t part = blockIdx.x;
    for (uint32_t back = blockIdx.y; back < uint32_t(x.rows); back += gridDim.y) {
        const uint32_t r = uint32_t(x.rows) - 1 - back;
        const Place at = place(x, r);
        const int64_t token = load_int(tokens, offset(tokens, at));
        T* g = grad + int64_t(r) * x.vocab;
        const T* row = row_of<T>(x, at);
        const Span span = span_of(row, x.vocab);
        const int from = int(part) * kGradVecs, t = threadIdx.x;
        T* to = g + span.head;
        auto zeros = [&] {
#pragma unroll
            for (int u = 0; u < kGradUnroll; ++u) {
                const int n = from + u * kThreads;
                if (n + t < span.vecs) store_vec(to, n, t, vec_t{0, 0, 0, 0});
            }
            if (part == 0 && int(threadIdx.x) < span.extra)
                g[extra_element<T>(span, threadIdx.x)] = narrow<T>(0.f);
        };
        if (token == ignore) {
            zeros();
            continue;
        }
        vec_t v[kGradUnroll];
#pragma unroll
        for (int u = 0; u < kGradUnroll; ++u) {
            const int n = from + u * kThreads;
            v[u] = n + t < span.vecs ? load_vec(row + span.head, n, t) : nothing<T>();
        }
        const float m = stats[2 * int64_t(r)], s = stats[2 * int64_t(r) + 1], inv_s = 1.f / s;
        const bool beyond = token < 0 || token >= x.vocab;
        const float a = beyond ? NAN : f * load_f32(coef, at);
        const float h = kEntropy ? f * load_f32(entropy_coef, at) : 0.f;
        // Nor does a row count that nothing depends on: outside all pairs, it may hold anything.  (It is loaded all the same:
        // with the question in front, every row's loads wait for its coefficient, 306 -> 312 us for 8192 x 50257 bf16 with
        // entropies and both directions.)
        if (a == 0.f && h == 0.f) {
            zeros();
            continue;
        }
        // a + h (log q + H) = b + h ln2 y
        const float b = kEntropy ? a + h * (entropy[r] - logf(s)) : a, hy = h * kLn2;
        auto value = [&](float xj, int j) {
            const float y = below(xj, m, x.c);
            const float q = __builtin_amdgcn_exp2f(y) * inv_s;
            return -q * (kEntropy ? b + hy * fmaxf(y, -1e30f) : b) + (j == token ? a : 0.f);
        };
#pragma unroll
        for (int u = 0; u < kGradUnroll; ++u) {
            const int n = from + u * kThreads, j = span.head + (n + t) * kVec<T>;
            float out[kVec<T>];
            unpack<T>(v[u], out);
#pragma unroll
            for (int k = 0; k < kVec<T>; ++k) out[k] = value(out[k], j + k);
            if (n + t < span.vecs) store_vec(to, n, t, pack<T>(out));
        }
        if (part == 0 && int(threadIdx.x) < span.extra) {
            const int j = extra_element<T>(span, threadIdx.x);
            g[j] = narrow<T>(value(widen(row[j]), j));
        }
    }
}

// ---- how many rows count, and of which sequence

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
    const Place at = place_of_thread(x, r);
    if (tokens.data && load_int(tokens, offset(tokens, at)) == ignore) return false;
    return load_mask(mask, at);
}

// count[i]: of the kCountRows rows from i kCountRows on, how many count; or, with sequences (lengths not NULL), whether
// any does of sequence i, and in lengths[] how many for each row of the sequence.
// A few bytes a row: 4 us, a launch's latency, for the rows of one count.  A sequence has a workgroup to itself, so long
// ones show: 64 of 1024 rows 7 us, 16 of 4096 21, one of 65536 111 (in front of 102 of the rows' kernel at 1003 bf16).
__global__ __launch_bounds__(kThreads) void count_kernel(Rows x, PerRow tokens, int64_t ignore, PerRow mask,
                                                         Sequences seqs, uint32_t items, int32_t* __restrict__ count,
                                                         float* __restrict__ lengths,
                                                         uint32_t* __restrict__ ticket) {
    __shared__ float lds[kWaves];
    const uint32_t item = row_of_block();
    if (item >= items) return;
    int64_t from = int64_t(item) * kCountRows, to = min(from + kCountRows, int64_t(x.rows));
    if (lengths) sequence_rows(seqs, x, item, &from, &to);
    int n = 0;
    for (int64_t r = from + threadIdx.x; r < to; r += kThreads) n += counts(x, tokens, ignore, mask, uint32_t(r));
    // below 2^24 a thread; exact as floats where the sum is, too, else the weight's last bit
    const float all = block_sum(Floats<1>{{float(n)}}, lds).v[0];
    if (threadIdx.x == 0) count[item] = lengths ? all > 0.f : int32_t(all);
    if (item == 0 && threadIdx.x == 0) *ticket = 0;
    if (lengths)
        for (int64_t r = from + threadIdx.x; r < to; r += kThreads) lengths[r] = all;
}

// The same for more than kCountGroups sequences: count[i] is how many of the i-th kCountGroups-th part of them have a row
// that counts.  A wave takes a sequence.
constexpr int kGroupThreads = 1024;
__global__ __launch_bounds__(kGroupThreads) void count_groups_kernel(Rows x, PerRow tokens, int64_t ignore, PerRow mask,
                                                                     Sequences seqs, int32_t* __restrict__ count,
                                                                     float* __restrict__ lengths,
                                                                     uint32_t* __restrict__ ticket) {
    constexpr int kGroupWaves = kGroupThreads / 64;
    __shared__ int with_any[kGroupWaves];
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    const int64_t each = (seqs.count + kCountGroups - 1) / kCountGroups;
    const int64_t first = blockIdx.x * each, end = min(first + each, seqs.count);
    int some = 0;
    for (int64_t i = first + wave; i < end; i += kGroupWaves) {
        int64_t from, to;
        sequence_rows(seqs, x, i, &from, &to);
        int n = 0;
        for (int64_t r = from + lane; r < to; r += 64) n += counts(x, tokens, ignore, mask, uint32_t(r));
        const float all = wave_sum(float(n));
        some += all > 0.f;
        for (int64_t r = from + lane; r < to; r += 64) lengths[r] = all;
    }
    if (lane == 0) with_any[wave] = some;
    __syncthreads();
    if (threadIdx.x == 0) {
        int all = 0;
        for (int w = 0; w < kGroupWaves; ++w) all += with_any[w];
        count[blockIdx.x] = all;
        if (blockIdx.x == 0) *ticket = 0;
    }
}

__global__ __launch_bounds__(kThreads) void zero_kernel(float* __restrict__ x, int64_t n) {
    const int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x;
    if (i < n) x[i] = 0.f;
}

// The sums of the rows' parts, always in the same order: of kResultRows a workgroup, and of the workgroups' by the last of
// them (65536 rows: 5 us; one workgroup alone took 21).
constexpr int kResultThreads = 1024;
constexpr int kResultRows = 4096;
__global__ __launch_bounds__(kResultThreads) void result_kernel(const float4* __restrict__ parts, uint32_t rows,
                                                                Result out) {
    __shared__ float lds[kResultThreads / 64 * 3];
    const uint32_t each = (rows + gridDim.x - 1) / gridDim.x, from = blockIdx.x * each;
    const uint32_t to = rows - from < each ? rows : from + each;
    Floats<3> sum = {{0.f, 0.f, 0.f}};
    for (uint32_t i = from + threadIdx.x; i < to; i += kResultThreads) {
        const float4 x = parts[i];
        sum.v[0] += x.x;
        sum.v[1] += x.y;
        sum.v[2] += x.z;
    }
    sum = block_sum<3, kResultThreads>(sum, lds);
    if (gridDim.x > 1) {
        put_part(out, blockIdx.x, sum.v[0], sum.v[1], sum.v[2]);
    } else if (threadIdx.x == 0) {
        out.result[0] = sum.v[0] * out.f;
        out.result[1] = sum.v[1];
        out.result[2] = sum.v[2];
    }
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

// The sum over the workgroup in 64 bits.
__device__ __forceinline__ double block_sum64(double x, double* lds) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o, 64);
    __syncthreads();
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = x;
    __syncthreads();
    x = lds[0];
    for (int w = 1; w < kWaves; ++w) x += lds[w];
    return x;
}

// One workgroup a pair: the sums over both sequences, the pair's loss and the rows' coefficients.  The sums are of a
// thousand log-probabilities, and what counts is how little they differ from a reference's: in 64 bits, as is the
// margin.  Latency alone: a sequence's offsets, then its rows' tokens and log-probabilities (8 pairs, 6000 rows: 8 us; 32
// pairs, 65536 rows: 13; one pair of them: 106).
__global__ __launch_bounds__(kThreads) void pairs_kernel(Rows x, Preference p, const float* __restrict__ row_logprobs,
                                                         float* __restrict__ logprobs, float* __restrict__ rewards,
                                                         Result out, float* __restrict__ coef) {
    __shared__ double lds[kWaves];
    const int64_t pairs = p.seqs.count / 2, i = row_of_block();
    if (i >= pairs) return;
    const PerRow none = {};
    int64_t from[2], to[2];
    double total[2], n[2], reward[2];
    for (int k = 0; k < 2; ++k) {
        sequence_rows(p.seqs, x, i + k * pairs, &from[k], &to[k]);
        double sum = 0.0;
        int count = 0;
        for (int64_t r = from[k] + threadIdx.x; r < to[k]; r += kThreads) {
            sum += row_logprobs[r];
            count += counts(x, p.tokens, p.ignore, none, uint32_t(r));
        }
        n[k] = p.length_average ? fmax(block_sum64(count, lds), 1.0) : 1.0;
        total[k] = block_sum64(sum, lds) / n[k];
        reward[k] = double(p.beta) * (total[k] - (p.ref ? p.ref[i + k * pairs] : 0.f));
    }
    const float h = float(reward[0] - reward[1]);
    float loss, slope;  // d loss / d h
    if (p.kind == MAMW_SIGMOID) {
        const float soft = log1pf(expf(-fabsf(h)));  // -log sigmoid(|h|)
        // h may be infinite (a token of no probability): what has no weight adds nothing
        loss = p.smoothing < 1.f ? (1.f - p.smoothing) * (soft + fmaxf(-h, 0.f)) : 0.f;
        if (p.smoothing > 0.f) loss += p.smoothing * (soft + fmaxf(h, 0.f));
        slope = p.smoothing - 1.f / (1.f + expf(h));
    } else if (p.kind == MAMW_IPO) {
        const float d = (h - 0.5f) / p.beta;
        loss = d * d;
        slope = 2.f * d / p.beta;
    } else {
        loss = h < 1.f ? 1.f - h : h >= 1.f ? 0.f : h;  // NaN stays
        slope = h < 1.f ? -1.f : h >= 1.f ? 0.f : h;
    }
    if (threadIdx.x < 2) {
        const int k = threadIdx.x;
        logprobs[i + k * pairs] = float(k ? total[1] : total[0]);
        rewards[i + k * pairs] = float(k ? reward[1] : reward[0]);
    }
    if (coef)
        for (int k = 0; k < 2; ++k) {
            const float c = (k ? -slope : slope) * p.beta / (float(pairs) * float(n[k]));
            for (int64_t r = from[k] + threadIdx.x; r < to[k]; r += kThreads) coef[r] = c;
        }
    put_part(out, uint32_t(i), loss, 0.f, 0.f);
}

// ---- launches

int launch_logprobs(const mamw_rows& x, const mamw_per_row& tokens, int64_t ignore, float temperature,
                    float* logprobs, float* entropy, float* stats, float* coef, uint32_t* ticket, hipStream_t stream) {
    const Rows rows = make_rows(x, temperature);
    // A gradient will read the rows again, the last ones first: as many as the memory-side cache has room for are left
    // in it.
    const double row = double(x.vocab) * (x.type == MAMW_F32 ? 4.0 : 2.0);
    const uint32_t keep_from = stats ? uint32_t(fmax(0.0, rows.rows - kKeptBytes / row)) : uint32_t(rows.rows);
    return with_type(x.type, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto n) {
            constexpr int kN = decltype(n)::value;
            return int(launch(K_OBJ_LOGPROBS, entropy ? 1 : 0, 0.0, row_bytes(x, false),
                              entropy ? logprobs_kernel<T, kN, true> : logprobs_kernel<T, kN, false>,
                              row_grid(rows.rows), dim3(kN), stream, rows, make_per_row(tokens), ignore,
                              logprobs, entropy, stats, coef, ticket, keep_from));
        };
        // By the vocabulary alone, so that a row's result does not depend on how many there are.
        const int64_t vecs = x.vocab / kVec<T>;
        if (vecs <= 512) return go(Int<64>());
        if (vecs <= 2048) return go(Int<256>());
        if (vecs <= 8192) return go(Int<512>());
        return go(Int<1024>());
    });
}

}  // namespace

int launch_count(const Rows& rows, const PerRow& tokens, int64_t ignore, const PerRow& mask, const Sequences& seqs,
                 const ObjectiveWorkspace& ws, bool by_sequence, char* base, hipStream_t stream) {
    if (by_sequence && seqs.offsets && rows.rows > 0) {
        const int st = int(launch(K_OBJ_COUNT, 1, 0.0, 0.0, zero_kernel, dim3(unsigned((rows.rows + kThreads - 1) / kThreads)),
                                  dim3(kThreads), stream, reinterpret_cast<float*>(base + ws.lengths_at),
                                  int64_t(rows.rows)));
        if (st != 0) return st;
    }
    uint32_t* ticket = reinterpret_cast<uint32_t*>(base + ws.ticket_at);
    if (ws.items == 0)
        return int(launch(K_OBJ_COUNT, 1, 0.0, 0.0, zero_kernel, dim3(1), dim3(kThreads), stream,
                          reinterpret_cast<float*>(ticket), int64_t(1)));
    if (by_sequence && seqs.count > kCountGroups)
        return int(launch(K_OBJ_COUNT, 2, 0.0, 0.0, count_groups_kernel, dim3(kCountGroups), dim3(kGroupThreads), stream, rows,
                          tokens, ignore, mask, seqs, reinterpret_cast<int32_t*>(base),
                          reinterpret_cast<float*>(base + ws.lengths_at), ticket));
    return int(launch(K_OBJ_COUNT, 0, 0.0, 0.0, count_kernel, row_grid(ws.items), dim3(kThreads), stream, rows,
                      tokens, ignore, mask, seqs, uint32_t(ws.items), reinterpret_cast<int32_t*>(base),
                      by_sequence ? reinterpret_cast<float*>(base + ws.lengths_at) : static_cast<float*>(nullptr),
                      ticket));
}

int launch_result(const Result& out, const ObjectiveWorkspace& ws, char* base, hipStream_t stream) {
    if (out.ticket) return MAMW_OK;
    Result sums = out;
    sums.parts = reinterpret_cast<float4*>(base + ws.ticket_at + 256);
    sums.ticket = reinterpret_cast<uint32_t*>(base + ws.ticket_at);
    sums.of = (out.of + kResultRows - 1) / kResultRows;
    if (sums.of > kResultBlocks) sums.of = kResultBlocks;
    if (sums.of == 0) sums.of = 1;
    return int(launch(K_OBJ_RESULT, 0, 0.0, 0.0, result_kernel, dim3(sums.of), dim3(kResultThreads), stream,
                      const_cast<const float4*>(out.parts), out.of, sums));
}

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
                           nullptr, nullptr, static_cast<hipStream_t>(stream));
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
        const unsigned parts = unsigned((logits->vocab / kVec<T> + kGradVecs - 1) / kGradVecs + (logits->vocab < kVec<T>));
        return int(launch(K_OBJ_GRAD, entropy_coef ? 1 : 0, 0.0, row_bytes(*logits, true),
                          entropy_coef ? logits_grad_kernel<T, true> : logits_grad_kernel<T, false>,
                          dim3(parts, unsigned(rows.rows < 65535 ? rows.rows : 65535)), dim3(kThreads),
                          static_cast<hipStream_t>(stream), rows, make_per_row(*tokens), ignore_index, stats,
                          make_per_row(*coef), entropy_coef ? make_per_row(*entropy_coef) : none, entropy, scale,
                          static_cast<T*>(grad)));
    });
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
    uint32_t* ticket = reinterpret_cast<uint32_t*>(base + ws.ticket_at);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    st = rows.rows > 0 ? launch_logprobs(*logits, p->tokens, p->ignore_index, p->temperature, row_logprobs, nullptr, stats,
                                         coef, ticket, s)
                       : int(launch(K_OBJ_COUNT, 1, 0.0, 0.0, zero_kernel, dim3(1), dim3(kThreads), s,
                                    reinterpret_cast<float*>(ticket), int64_t(1)));
    if (st != MAMW_OK) return st;
    const int64_t pairs = p->sequences / 2;
    const Result out = make_result(ws, base, pairs, true, 1.f / float(pairs), result);
    Preference d;
    d.tokens = make_per_row(p->tokens);
    d.ignore = p->ignore_index;
    d.ref = p->ref_logprobs;
    d.seqs = {p->offsets, p->sequences};
    d.beta = p->beta;
    d.smoothing = p->smoothing;
    d.kind = p->kind;
    d.length_average = p->length_average;
    if ((st = int(launch(K_OBJ_PAIRS, 0, 0.0, 0.0, pairs_kernel, row_grid(pairs), dim3(kThreads), s, rows, d,
                         static_cast<const float*>(row_logprobs), logprobs, rewards, out, coef))) != 0)
        return st;
    return launch_result(out, ws, base, s);
}
