// Distillation from a teacher's top logits for gfx950: the teacher's entries of all rows first, then the divergence of
// a row and its gradient in one pass.
#include "mamw_rows.h"

namespace mamw {
namespace {

// ---- the teacher's entries

struct TeacherArgs {
    PerRow logits, indices, lse, mask;
    int k;
};

__device__ __forceinline__ float load_float(const PerRow& a, int64_t i) {
    if (a.type == MAMW_F32) return reinterpret_cast<const float*>(a.data)[i];
    if (a.type == MAMW_BF16) return widen(reinterpret_cast<const bf16_t*>(a.data)[i]);
    return widen(reinterpret_cast<const _Float16*>(a.data)[i]);
}

constexpr int kPadding = -1;

// What the student's pass needs of a row's teacher: for each entry its index (kPadding: left out) and probability, and
struct TeacherRow {
    float sum_p, plogp;  // sum of p and of p log p
    int entries;         // different ones
    int beyond;          // some are outside the vocabulary
};
static_assert(sizeof(TeacherRow) == 16, "one 16-byte load a row");

// One wave a row, kTeacherRows rows a workgroup; entry k of the row is entry k / 64 of lane k % 64.  By itself, in
// front of the student's pass: there it would be one wave's chain of dependent steps while fifteen wait for it, once
// a row (128 entries: 16 us of 181 for 2048 rows of 128256 bf16, before later steps).
//
// An index that is given more than once becomes one entry with the sum of the probabilities.  A table of 2^14 bits
// finds those that may be: an entry whose bit is set already, by its own index or by another that falls on it, is
// compared with all others.
//
// p_k = exp(t_k / T - lse): with lse the logsumexp of the row's entries or the one that was given.  Latency: 6 us for
// 4096 rows of 128, 25 for 65536 of 64.
constexpr int kSeenBits = 1 << 14;

template <int kPerLane, bool kTail>
__global__ __launch_bounds__(64 * kTeacherRows) void teacher_kernel(Rows x, TeacherArgs a, int32_t* __restrict__ index,
                                                                    float* __restrict__ probs,
                                                                    TeacherRow* __restrict__ info, uint32_t groups,
                                                                    uint32_t items, int32_t* __restrict__ count,
                                                                    uint32_t* __restrict__ ticket) {
    __shared__ uint32_t seen_bits[kTeacherRows][kSeenBits / 32];
    __shared__ int counted[kTeacherRows];
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    const uint32_t group = row_of_block();
    if (group >= groups) return;
    // The first workgroups count, too: a row a thread.
    static_assert(64 * kTeacherRows == kCountRows, "one row a thread");
    const int64_t of_thread = int64_t(group) * kCountRows + threadIdx.x;
    const bool counts_ = group < items && of_thread < x.rows && load_mask(a.mask, place_of_thread(x, uint32_t(of_thread)));
    const int64_t r = int64_t(group) * kTeacherRows + __builtin_amdgcn_readfirstlane(wave);
    if (r < x.rows) {
        const Place at = place(x, uint32_t(r));
        if (load_mask(a.mask, at)) {
            uint32_t* seen = seen_bits[wave];
#pragma unroll
            for (int i = 0; i < kSeenBits / 32 / 64; ++i) seen[i * 64 + lane] = 0;
            const int64_t tl = offset(a.logits, at), ti = offset(a.indices, at);
            int32_t idx[kPerLane];
            float t[kPerLane];
            bool beyond = false;
            float top = -INFINITY;
#pragma unroll
            for (int e = 0; e < kPerLane; ++e) {
                const int k = e * 64 + lane;
                const bool is = k < a.k;
                t[e] = is ? load_float(a.logits, tl + k) : -INFINITY;
                const int64_t j = is ? load_int(a.indices, ti + k) : -1;
                const bool given = j >= 0 && t[e] != -INFINITY, in = given && j < x.vocab;
                beyond |= given && !in;
                idx[e] = in ? int32_t(j) : kPadding;
                if (in) top = fmaxf(top, t[e]);
            }
            float shift;
            if constexpr (kTail) {
                top = 0.f;
                shift = load_f32(a.lse, at);
            } else {
                top = wave_max(top);
                float z = 0.f;
#pragma unroll
                for (int e = 0; e < kPerLane; ++e)
                    if (idx[e] >= 0) z += __builtin_amdgcn_exp2f(below(t[e], top, x.c));
                shift = logf(wave_sum(z));
            }
            float sum_p = 0.f, plogp = 0.f;
#pragma unroll
            for (int e = 0; e < kPerLane; ++e) {
                if (idx[e] < 0) continue;
                const float l = (t[e] - top) * x.inv_t - shift, p = expf(l);
                sum_p += p;
                plogp += p > 0.f ? p * l : p;  // p log p = 0 at p = 0; NaN stays
                t[e] = p;
            }
            sum_p = wave_sum(sum_p);
            plogp = wave_sum(plogp);
            // the bits of one wave are its own: its LDS accesses stay in order
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            uint64_t again[kPerLane];
#pragma unroll
            for (int e = 0; e < kPerLane; ++e) {
                const uint32_t h = uint32_t(idx[e]) % kSeenBits, bit = 1u << (h & 31);
                again[e] = __ballot(idx[e] >= 0 && (atomicOr(&seen[h >> 5], bit) & bit));
            }
#pragma unroll
            for (int e = 0; e < kPerLane; ++e)
                while (again[e]) {
                    const int l = __builtin_ctzll(again[e]);
                    again[e] &= again[e] - 1;
                    const int j = __builtin_amdgcn_readlane(idx[e], l);
                    if (j < 0) continue;  // made one with an earlier entry meanwhile
                    float p = 0.f;
#pragma unroll
                    for (int i = 0; i < kPerLane; ++i) p += idx[i] == j ? t[i] : 0.f;
                    p = wave_sum(p);
                    bool found = false;
#pragma unroll
                    for (int i = 0; i < kPerLane; ++i) {
                        const uint64_t same = __ballot(idx[i] == j);
                        if (idx[i] == j) {
                            const bool first = !found && lane == __builtin_ctzll(same);
                            t[i] = p;
                            idx[i] = first ? j : kPadding;
                        }
                        found |= same != 0;
                    }
                }
            int entries = 0;
#pragma unroll
            for (int e = 0; e < kPerLane; ++e) {
                const int k = e * 64 + lane;
                entries += __popcll(__ballot(idx[e] >= 0));
                if (k < a.k) {
                    index[r * a.k + k] = idx[e];
                    probs[r * a.k + k] = t[e];
                }
            }
            const bool any_beyond = __any(beyond);
            if (lane == 0) info[r] = {sum_p, plogp, entries, any_beyond};
        }
    }
    if (group >= items) return;
    const int n = __popcll(__ballot(counts_));
    if (lane == 0) counted[wave] = n;
    __syncthreads();
    if (threadIdx.x == 0) {
        int all = 0;
        for (int w = 0; w < kTeacherRows; ++w) all += counted[w];
        count[group] = all;
        if (group == 0) *ticket = 0;
    }
}

// ---- the student's rows

struct Distill {
    PerRow mask;
    int64_t items;
    int k;
    float temperature, scale;
    const int32_t* count;
    const int32_t* index;
    const float* probs;
    const TeacherRow* info;
};

// A wave's part of a row: its statistics (kTail: without the teacher's entries); of those entries alone the largest
// logit `top` and, below it, the sum s_in of 2^y; the sum p of their probabilities and px of p (x - top).
struct Parts {
    float m, s, top, s_in, p, px;
};

// 2^y of `from` below a larger `to`; finite, for sums that are 0.
__device__ __forceinline__ float factor(float from, float to, float c) {
    return __builtin_amdgcn_exp2f(below(from, reference(to), c));
}

// p (from - to): nothing where p is, however far apart the two.
__device__ __forceinline__ float moved(float p, float from, float to) {
    return p == 0.f ? 0.f : p * (reference(from) - reference(to));
}

// p (x - top) goes by the entries' own largest logit: a wave may see nothing but the type's lowest value in the row, and
// a difference to that would have lost x.  (p is the wave's afterwards, too.)
template <int kThreads_, bool kTail>
__device__ __forceinline__ Parts parts_over_block(Parts mine, float c, Parts* lds) {
    constexpr int kN = kThreads_ / 64;
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = mine;
    __syncthreads();
    mine = lds[threadIdx.x % kN];
    float m = mine.m, top = mine.top;
#pragma unroll
    for (int o = kN / 2; o >= 1; o >>= 1) {
        m = fmaxf(m, __shfl_xor(m, o, 64));
        top = fmaxf(top, __shfl_xor(top, o, 64));
    }
    mine.s *= factor(mine.m, m, c);
    if (kTail) mine.s_in *= factor(mine.top, top, c);
    mine.px += moved(mine.p, mine.top, top);
#pragma unroll
    for (int o = kN / 2; o >= 1; o >>= 1) {
        mine.s += __shfl_xor(mine.s, o, 64);
        if (kTail) mine.s_in += __shfl_xor(mine.s_in, o, 64);
        mine.px += __shfl_xor(mine.px, o, 64);
    }
    mine.m = m;
    mine.top = top;
    return mine;
}

// The teacher's entries of a row that are to be left out of its sum, marked in LDS: a byte for each held vector, all
// bytes of a thread together, so that it reads them at once (a bit for each element of the vocabulary, looked up for
// every vector, took 30 us of 178 for 2048 rows of 128256 bf16); a bit for each single element; with kRest a bit for
// each element of the vocabulary, looked at for the vectors that are not held.
template <typename T, int kThreads_, int kVecs, bool kRest>
struct Marks {
    static constexpr int kWords = (kVecs + 3) / 4;  // of a thread
    static constexpr int kHeld = kThreads_ * kWords;

    static constexpr int kSingles = (kExtra + 31) / 32;
    static constexpr int kTable = kHeld + kSingles;  // where the bits of all elements begin

    static __host__ __device__ constexpr int words(int vocab) { return kTable + (kRest ? (vocab + 31) / 32 : 0); }

    // Marks element j, if `wave` is the wave that holds it, or -1.
    static __device__ __forceinline__ void set(uint32_t* table, const Span& s, int j, int wave) {
        const int n = j < s.head ? -1 : (j - s.head) / kVec<T>;
        const bool is_single = n < 0 || n >= s.vecs;
        const int single = j < s.head ? j : j - s.vecs * kVec<T>;
        if (wave >= 0 && wave != (is_single ? single / 64 : n % kThreads_ / 64)) return;
        if (is_single) {
            atomicOr(&table[kHeld + single / 32], 1u << (single & 31));
        } else if (n < kVecs * kThreads_) {
            const int i = n / kThreads_, k = (j - s.head) % kVec<T>;
            atomicOr(&table[n % kThreads_ * kWords + i / 4], 1u << (i % 4 * 8 + k));
        } else {
            atomicOr(&table[kTable + (j >> 5)], 1u << (j & 31));
        }
    }

    // The elements of v whose bits are set become nothing.
    static __device__ __forceinline__ void leave_out(vec_t& v, uint32_t bits) {
        const vec_t none = nothing<T>();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) {
                const uint32_t m = uint32_t(__builtin_amdgcn_sbfe(int32_t(bits), i, 1));
                v[i] = (v[i] & ~m) | (none[i] & m);
            } else {
                const uint32_t lo = uint32_t(__builtin_amdgcn_sbfe(int32_t(bits), 2 * i, 1)) & 0xffffu;
                const uint32_t hi = uint32_t(__builtin_amdgcn_sbfe(int32_t(bits), 2 * i + 1, 1)) & 0xffff0000u;
                v[i] = (v[i] & ~(lo | hi)) | (none[i] & (lo | hi));
            }
        }
    }

    // The bits of vector n, not held: elements head + n kVec and on.
    static __device__ __forceinline__ uint32_t rest(const uint32_t* table, const Span& s, int n, int vocab) {
        const int j = s.head + n * kVec<T>, w = j >> 5;
        uint32_t m = table[kTable + w] >> (j & 31);
        if ((j & 31) + kVec<T> > 32 && w + 1 < (vocab + 31) / 32) m |= table[kTable + 1 + w] << (32 - (j & 31));
        return m & ((1u << kVec<T>) - 1u);
    }
};

// loss = sum p (log p - log q), with kTail + P log(P / Q), where P and Q are what the teacher and the student leave to
// all other elements; g_j = w (q_j A - p_j), and for those others w q_j (A - P / Q), with A = sum p + P.  That is 1, but for
// probabilities that add up to more than 1 (logits rounded after their lse was taken; P is at least 2^-20 then), and
// to less where there are no others.
//
// kTail: the teacher's entries are taken out of the row and their sum is added from the gathered logits, so that the
// sum over all others is not the small difference of two large ones.
//
// One read and one write, as in the policy's kernel: 4096 x 128256 bf16 with 128 entries and a rest, 2409 rows that
// count, 0.62 GB read and 1.05 written in 325 us, 5.1 TB/s; 2048 x 50257 fp32 with 64 entries, 0.14 and 0.41 GB, in 99,
// 5.6 TB/s.  Writing the entries over what the row's vectors left is 4 of these 325 us and as many as 20 to 28 of the 222
// of 65536 x 4000 bf16 with 64 entries, 35592 rows that count; the gathers of the entries' logits are 14 there.
template <typename T, int kThreads_, int kVecs, bool kRest, bool kTail>
__global__ __launch_bounds__(kThreads_, kRowWaves<kVecs>) void distill_kernel(
    Rows x, Distill p, Result out, const float* __restrict__ scale, int unless_one,
    T* __restrict__ grad) {
    extern __shared__ uint32_t marked[];
    __shared__ Parts lds[kThreads_ / 64];
    constexpr int kEntries = MAMW_MAX_TEACHER / kThreads_;  // of a thread
    const float f = scale ? *scale : 1.f;
    if (scale && unless_one && f == 1.f) return;
    const uint32_t r = row_of_block();
    if (r >= uint32_t(x.rows)) return;
    const Place at = place(x, r);
    T* g = grad ? grad + int64_t(r) * x.vocab : nullptr;
    if (!load_mask(p.mask, at)) {
        if (g) zero_row(g, x.vocab, kThreads_);
        put_part(out, r, 0.f, 0.f, 0.f);
        return;
    }
    const T* row = row_of<T>(x, at);
    // The entries' indices before the row, to mark them while it is on its way; the logits they point to behind it, to be
    // looked at where it has been waited for anyway.
    int32_t index[kEntries];
    float probs[kEntries];
    Raw<T> xs[kEntries];
#pragma unroll
    for (int e = 0; e < kEntries; ++e) {
        const int k = e * kThreads_ + int(threadIdx.x);
        index[e] = kPadding;
        probs[e] = 0.f;
        if (k < p.k) {
            index[e] = p.index[int64_t(r) * p.k + k];
            probs[e] = p.probs[int64_t(r) * p.k + k];
        }
    }
    constexpr int kAhead = kTail && !kRest ? 4 : 0;  // of all entries, by each wave
    int32_t ahead[kAhead + 1];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
        ahead[i] = p.index[int64_t(r) * p.k + min(i * 64 + int(threadIdx.x % 64), p.k - 1)];
    const TeacherRow teacher = p.info[r];
    const Counts counted(p.count, p.items);
    HeldRow<T, kThreads_, kVecs, kRest> held;
    held.load(row, x.vocab, p.count);
    using Mark = Marks<T, kThreads_, kVecs, kRest>;
    if constexpr (kTail && !kRest) {
        // Every wave by itself looks through all entries for those in its own vectors: with a barrier here no wave begins
        // before the last one has started, behind the workgroup before (2048 rows of 128256 bf16: 17 us of 178).
        const int wave = threadIdx.x / 64;
#pragma unroll
        for (int i = 0; i < Mark::kWords; ++i) marked[int(threadIdx.x) * Mark::kWords + i] = 0;
        // single element e is thread e's: two words of wave 0, one of wave 1
        if (threadIdx.x % 32 == 0 && int(threadIdx.x) < 32 * Mark::kSingles) marked[Mark::kHeld + threadIdx.x / 32] = 0;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (ahead[i] >= 0 && i * 64 < p.k) Mark::set(marked, held.span, ahead[i], wave);
#pragma unroll 1
        for (int k = kAhead * 64 + int(threadIdx.x % 64); k < p.k; k += 64) {
            const int j = p.index[int64_t(r) * p.k + k];
            if (j >= 0) Mark::set(marked, held.span, j, wave);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    } else if constexpr (kTail) {
        for (int j = threadIdx.x; j < Mark::words(x.vocab); j += kThreads_) marked[j] = 0;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kEntries; ++e)
            if (index[e] >= 0) Mark::set(marked, held.span, index[e], -1);
        __syncthreads();
    }
#pragma unroll
    for (int e = 0; e < kEntries; ++e) xs[e] = raw_at(row + max(index[e], 0));
    uint32_t mine[Mark::kWords] = {};
    if constexpr (kTail) {
#pragma unroll
        for (int i = 0; i < Mark::kWords; ++i) mine[i] = marked[int(threadIdx.x) * Mark::kWords + i];
        if (held.has_single() && (marked[Mark::kHeld + threadIdx.x / 32] >> (threadIdx.x & 31) & 1u)) held.single_ = raw_nothing<T>();
    }
    auto hold = [&](vec_t& v, int i) {
        if constexpr (kTail) {
            const uint32_t bits = mine[i / 4] >> (i % 4 * 8) & 0xffu;
            if (__any(bits != 0)) Mark::leave_out(v, bits);
        }
    };
    auto change = [&](vec_t& v, int n) {
        if constexpr (kTail && kRest)
            if (n < held.span.vecs) {
                const uint32_t bits = Mark::rest(marked, held.span, n, x.vocab);
                if (bits) Mark::leave_out(v, bits);
            }
    };
    Stats st = held.stats(x.c, hold, change);
    // Both maxima over the wave, then all sums, side by side, and no more of the entries' slots than k fills: with
    // one after the other 65536 x 1003 bf16 took 131 us instead of 130, 134 instead of 133 with a rest.
    float m_wave = st.m, top = -INFINITY;
#pragma unroll
    for (int e = 0; e < kEntries; ++e)
        if (e * kThreads_ < p.k && index[e] >= 0) top = fmaxf(top, xs[e].value());
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        m_wave = fmaxf(m_wave, __shfl_xor(m_wave, o, 64));
        top = fmaxf(top, __shfl_xor(top, o, 64));
    }
    move_to<false>(st, m_wave, x.c);
    const float ref_top = reference(top);
    float s_wave = st.s, s_in = 0.f, sum_p = 0.f, px_in = 0.f;
#pragma unroll
    for (int e = 0; e < kEntries; ++e) {
        if (e * kThreads_ >= p.k || index[e] < 0) continue;
        if (kTail) s_in += __builtin_amdgcn_exp2f(below(xs[e].value(), ref_top, x.c));
        sum_p += probs[e];
        px_in += probs[e] > 0.f ? probs[e] * (xs[e].value() - ref_top) : probs[e];  // 0 * -inf; NaN stays
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        s_wave += __shfl_xor(s_wave, o, 64);
        if (kTail) s_in += __shfl_xor(s_in, o, 64);
        sum_p += __shfl_xor(sum_p, o, 64);
        px_in += __shfl_xor(px_in, o, 64);
    }
    const Parts all_parts = parts_over_block<kThreads_, kTail>({m_wave, s_wave, top, s_in, sum_p, px_in}, x.c, lds);
    // m, rest: of what the row holds; all, s: with the teacher's entries
    const float m = all_parts.m, rest = all_parts.s, all = kTail ? fmaxf(m, all_parts.top) : m;
    const float m_to_all = kTail ? factor(m, all, x.c) : 1.f;
    const float s = kTail ? rest * m_to_all + all_parts.s_in * factor(all_parts.top, all, x.c) : rest, inv_s = 1.f / s;
    // sum p (log p - log q), with log q = (x - all) / T - log s
    const float px = all_parts.px + moved(teacher.sum_p, all_parts.top, all);
    float loss = teacher.entries > 0 ? teacher.plogp - px * x.inv_t + teacher.sum_p * logf(s) : 0.f;
    float in = teacher.entries > 0 ? 1.f : 0.f;  // times inv_s 2^y: A q_j
    float outside = in * inv_s;                  // times 2^y below m: A q_j - P q_j / Q, outside the entries
    if constexpr (kTail) {
        in = teacher.sum_p;
        if (teacher.entries < x.vocab) {
            // Q = rest 2^(m below all) / s may be beyond what 32 bits hold, its logarithm and q_j / Q = 2^y / rest are not
            const float rest_p = fmaxf(1.f - teacher.sum_p, kSmallestTail);
            loss += rest_p * (logf(rest_p * s / rest) + (all - m) * x.inv_t);
            in += rest_p;
            outside = in * m_to_all * inv_s - rest_p / rest;
        }
    }
    const float count = counted.all();
    if (g) {
        const float w = teacher.beyond ? NAN : f * p.scale * p.temperature / count;
        held.write(g, w * outside, m, x.c, change);
        __syncthreads();  // then the entries themselves, over what was written there
#pragma unroll
        for (int e = 0; e < kEntries; ++e)
            if (index[e] >= 0)
                g[index[e]] = narrow<T>(w * (in * inv_s * __builtin_amdgcn_exp2f(below(xs[e].value(), all, x.c)) - probs[e]));
    }
    put_part(out, r, (teacher.beyond ? NAN : loss) / count, 0.f, 0.f);
}

// ---- launches

struct DistillWorkspace {
    int32_t* count;
    uint32_t* ticket;
    int32_t* index;
    float* probs;
    TeacherRow* info;
};

DistillWorkspace parts_of(const ObjectiveWorkspace& ws, char* base, int64_t rows, int64_t k) {
    DistillWorkspace w;
    w.count = reinterpret_cast<int32_t*>(base);
    w.ticket = reinterpret_cast<uint32_t*>(base + ws.ticket_at);
    w.index = reinterpret_cast<int32_t*>(base + ws.lengths_at);
    w.probs = reinterpret_cast<float*>(w.index + rows * k);
    w.info = reinterpret_cast<TeacherRow*>(reinterpret_cast<float4*>(base + ws.partials_at) + rows);
    return w;
}

int launch_teacher(const mamw_rows& x, const mamw_distill& p, const ObjectiveWorkspace& ws, const DistillWorkspace& w,
                   hipStream_t stream) {
    const Rows rows = make_rows(x, p.temperature);
    if (rows.rows == 0) return MAMW_OK;
    const TeacherArgs a = {make_per_row(p.teacher_logits), make_per_row(p.teacher_indices),
                           make_per_row(p.teacher_lse), make_per_row(p.mask), int(p.k)};
    const int64_t groups = (int64_t(rows.rows) + kTeacherRows - 1) / kTeacherRows;
    auto go = [&](auto n) {
        constexpr int kPerLane = decltype(n)::value;
        return int(launch(K_OBJ_TEACHER, kPerLane, 0.0, 0.0,
                          p.teacher_lse.data ? teacher_kernel<kPerLane, true> : teacher_kernel<kPerLane, false>,
                          row_grid(groups), dim3(64 * kTeacherRows), stream, rows, a, w.index, w.probs, w.info,
                          uint32_t(groups), uint32_t(ws.items), w.count, w.ticket));
    };
    return p.k <= 64 ? go(Int<1>()) : p.k <= 128 ? go(Int<2>()) : p.k <= 256 ? go(Int<4>())
         : p.k <= 512 ? go(Int<8>()) : go(Int<16>());
}

int launch_distill(const mamw_rows& x, const mamw_distill& p, const ObjectiveWorkspace& ws, const DistillWorkspace& w,
                   const Result& out, const float* scale, int unless_one, void* grad, hipStream_t stream) {
    const Rows rows = make_rows(x, p.temperature);
    if (rows.rows == 0) return MAMW_OK;
    Distill d;
    d.mask = make_per_row(p.mask);
    d.items = ws.items;
    d.k = int(p.k);
    d.temperature = p.temperature;
    d.scale = p.scale;
    d.count = w.count;
    d.index = w.index;
    d.probs = w.probs;
    d.info = w.info;
    const bool tail = p.teacher_lse.data != nullptr;
    return with_type(x.type, [&](auto t) {
        using T = decltype(t);
        return with_held_row<true>(x.vocab / kVec<T>, [&](auto n, auto v, auto rest) {
            constexpr int kN = decltype(n)::value, kV = decltype(v)::value;
            constexpr bool kRest = decltype(rest)::value != 0;
            const size_t lds = tail ? size_t(Marks<T, kN, kV, kRest>::words(int(x.vocab))) * 4 : 0;
            return int(launch_lds(K_OBJ_DISTILL, kN + tail, 0.0, row_bytes(x, grad != nullptr),
                                  tail ? distill_kernel<T, kN, kV, kRest, true> : distill_kernel<T, kN, kV, kRest, false>,
                                  row_grid(rows.rows), dim3(kN), lds, stream, rows, d, out, scale,
                                  unless_one, static_cast<T*>(grad)));
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
    const int64_t rows = logits->outer * logits->inner;
    char* base = static_cast<char*>(workspace);
    const DistillWorkspace w = parts_of(ws, base, rows, p->k);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if ((st = launch_teacher(*logits, *p, ws, w, s)) != MAMW_OK) return st;
    const Result out = make_result(ws, base, rows, rows > 0, p->scale * p->temperature * p->temperature, result);
    if ((st = launch_distill(*logits, *p, ws, w, out, nullptr, 0, grad, s)) != MAMW_OK) return st;
    return launch_result(out, ws, base, s);
}

extern "C" int mamw_distill_grad(const mamw_rows* logits, const mamw_distill* p, const float* scale, int unless_one,
                                 void* grad, void* workspace, size_t workspace_bytes, mamw_stream_t stream) {
    ObjectiveWorkspace ws;
    int st = check_distill(logits, p, grad, &ws);
    if (st != MAMW_OK) return st;
    if ((st = check_workspace(ws, workspace, workspace_bytes)) != MAMW_OK) return st;
    const int64_t rows = logits->outer * logits->inner;
    if (!scale || (!grad && rows > 0)) return MAMW_ERR_NULL;
    const DistillWorkspace w = parts_of(ws, static_cast<char*>(workspace), rows, p->k);
    return launch_distill(*logits, *p, ws, w, Result(), scale, unless_one, grad, static_cast<hipStream_t>(stream));
}
