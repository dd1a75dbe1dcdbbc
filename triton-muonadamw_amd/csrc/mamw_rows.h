// Device side of the objectives' kernels over rows of logits: element types, where a row and what goes with it lie,
// the statistics of its softmax, and a row held in registers.
#pragma once

#include "mamw_device.h"
#include "mamw_launch.h"
#include "mamw_objectives.h"

namespace mamw {

constexpr int kThreads = 256;  // of the kernels that are not over logits
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

// An element as it was loaded, in a register of its own: a value that is not looked at yet is not waited for.
template <typename T>
struct Raw {
    uint32_t bits;
    __device__ __forceinline__ float value() const {
        if constexpr (sizeof(T) == 4)
            return __uint_as_float(bits);
        else if constexpr (__is_same(T, bf16_t))
            return bf16_to_f32(bits);
        else
            return float(__builtin_bit_cast(_Float16, uint16_t(bits)));
    }
};
template <typename T>
__device__ __forceinline__ Raw<T> raw_at(const T* x) {
    if constexpr (sizeof(T) == 4)
        return {*reinterpret_cast<const uint32_t*>(x)};
    else
        return {*reinterpret_cast<const uint16_t*>(x)};
}
template <typename T>
__device__ __forceinline__ Raw<T> raw_nothing() {
    return {sizeof(T) == 4 ? 0xff800000u : __is_same(T, bf16_t) ? 0xff80u : 0xfc00u};
}

// 16 bytes of a row: kVec<T> elements.
typedef uint32_t vec_t __attribute__((ext_vector_type(4)));
typedef vec_t any_vec_t __attribute__((aligned(2)));  // at any element
template <typename T>
constexpr int kVec = int(16 / sizeof(T));

template <typename T>
__device__ __forceinline__ void unpack(vec_t v, float* f) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(v[i]);
    } else if constexpr (__is_same(T, bf16_t)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(v[i] << 16);
            f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = float(__builtin_bit_cast(_Float16, uint16_t(v[i] & 0xffffu)));
            f[2 * i + 1] = float(__builtin_bit_cast(_Float16, uint16_t(v[i] >> 16)));
        }
    }
}

template <typename T>
__device__ __forceinline__ vec_t pack(const float* f) {
    vec_t v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4)
            v[i] = __float_as_uint(f[i]);
        else if constexpr (__is_same(T, bf16_t))
            v[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
        else
            v[i] = uint32_t(__builtin_bit_cast(uint16_t, _Float16(f[2 * i]))) |
                   uint32_t(__builtin_bit_cast(uint16_t, _Float16(f[2 * i + 1]))) << 16;
    }
    return v;
}

// Elements of no probability.
template <typename T>
__device__ __forceinline__ vec_t nothing() {
    const uint32_t w = sizeof(T) == 4 ? 0xff800000u : __is_same(T, bf16_t) ? 0xff80ff80u : 0xfc00fc00u;
    return {w, w, w, w};
}

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

// Row r is the same for the whole workgroup; so that addresses made of it stay in scalar registers, the quotient, which
// the vector unit forms, is brought back there.
__device__ __forceinline__ Place place(const Rows& x, uint32_t r) {
    const uint32_t o = __builtin_amdgcn_readfirstlane(r / x.inner);
    return {o, r - o * x.inner};
}
__device__ __forceinline__ uint32_t row_of_block() { return blockIdx.y * gridDim.x + blockIdx.x; }
// The same for rows that differ between threads.
__device__ __forceinline__ Place place_of_thread(const Rows& x, uint32_t r) {
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

struct Sequences {
    const int64_t* offsets;
    int64_t count;
};

// ---- reductions over the workgroup, always in the same order

template <int N>
struct Floats {
    float v[N];
};

template <int N, int kThreads_ = kThreads>
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
        for (int w = 1; w < kThreads_ / 64; ++w) x.v[i] += lds[w * N + i];
    }
    return x;
}

// ---- a row

// y_j = log2 of exp((x_j - m) / T).  The difference first: logits and masks may be the type's lowest value, whose
// product with log2(e) / T overflows.  (The fused form, one operation less, is as fast where memory is the bound: 590
// against 586 us for a policy loss over 8192 x 128256 bf16; 319 against 325 for a distillation over 4096 of them.)
__device__ __forceinline__ float below(float x, float m, float c) { return (x - m) * c; }

// A row as `vecs` vectors of 16 bytes from the first 128-byte boundary on, at element `head`, and `extra` single
// elements before and after them, at most kExtra.  A wave's 64 vectors are whole lines of the cache then.  Loads that
// straddle 16 bytes cost: 8192 x 50257 bf16 with its odd rows took 162 us to read, against 117 for as many bytes on the
// boundary; stores that share lines, too (4096 x 50257 fp32 with its gradient: 234 us from the first 16-byte boundary,
// 212 from the first of 64, 207 of 128, 207 of 256).
struct Span {
    int head, vecs, extra;
};
constexpr uintptr_t kLine = 128;
constexpr int kExtra = 63 + 7;

template <typename T>
__device__ __forceinline__ Span span_of(const T* row, int vocab) {
    Span s;
    s.head = min(vocab, int((-reinterpret_cast<uintptr_t>(row) & (kLine - 1)) / sizeof(T)));
    s.vecs = (vocab - s.head) / kVec<T>;
    s.extra = s.head + (vocab - s.head) % kVec<T>;
    return s;
}

// The element of single element e < extra.
template <typename T>
__device__ __forceinline__ int extra_element(const Span& s, int e) {
    return e < s.head ? e : e + s.vecs * kVec<T>;
}

// The thread of `threads` that writes element j, where vector n is thread n % threads' and single element e thread e's
// (there are more threads than kExtra).
template <typename T>
__device__ __forceinline__ int owner_of(const Span& s, int j, int threads) {
    if (j < s.head) return j;
    const int n = (j - s.head) / kVec<T>;
    return n < s.vecs ? n % threads : j - s.vecs * kVec<T>;
}

// Rows pass through once: kept out of the caches' way (8192 x 128256 bf16 and their gradient: 620 us with ordinary
// loads and stores, 586 with these; the log-probabilities of 8192 x 50257 bf16: 94 and 83).
//
// Vector `thread` of those from `first` on, with `first` the same for the whole workgroup: scalar address and 32-bit
// offset, no registers for sixteen 64-bit addresses.
// kKeep: through the caches all the same, for who reads the row next.
template <bool kKeep = false>
__device__ __forceinline__ vec_t load_vec(const void* vecs, int first, int thread) {
    const char* at = static_cast<const char*>(vecs) + int64_t(first) * 16;
    const vec_t* from = reinterpret_cast<const vec_t*>(at + uint32_t(thread) * 16u);
    if constexpr (kKeep)
        return *from;
    else
        return __builtin_nontemporal_load(from);
}
__device__ __forceinline__ void store_vec(void* vecs, int first, int thread, vec_t v) {
    // at any element: the gradient's rows may lie otherwise than the logits'
    char* at = static_cast<char*>(vecs) + int64_t(first) * 16;
    __builtin_nontemporal_store(v, reinterpret_cast<any_vec_t*>(at + uint32_t(thread) * 16u));
}

template <typename T>
__device__ __forceinline__ void zero_row(T* __restrict__ g, int vocab, int threads) {
    const Span s = span_of(g, vocab);
    const int t = threadIdx.x;
    for (int n = 0; n + t < s.vecs; n += threads) store_vec(g + s.head, n, t, vec_t{0, 0, 0, 0});
    if (int(threadIdx.x) < s.extra) g[extra_element<T>(s, threadIdx.x)] = narrow<T>(0.f);
}

// The logit of the row's token, on its way.
template <typename T>
struct Chosen {
    bool beyond;  // the vocabulary
    Raw<T> raw;

    __device__ __forceinline__ Chosen(const T* row, int64_t token, int vocab)
        : beyond(token < 0 || token >= vocab), raw(raw_at(row + (beyond ? 0 : token))) {}
    __device__ __forceinline__ float value() const { return beyond ? NAN : raw.value(); }
};

// Running softmax statistics: the largest logit m so far, s = sum of 2^y and sy = sum of 2^y y (entropies) below it.
struct Stats {
    float m, s, sy;
};
__device__ __forceinline__ Stats no_stats() { return {-INFINITY, 0.f, 0.f}; }

__device__ __forceinline__ float reference(float m) { return m == -INFINITY ? 0.f : m; }

// st as seen from a larger m.
template <bool kEntropy>
__device__ __forceinline__ void move_to(Stats& st, float m, float c) {
    const float y = fmaxf(below(st.m, reference(m), c), -1e30f);  // finite: times s = 0 it is 0
    const float f = __builtin_amdgcn_exp2f(y);
    if (kEntropy) st.sy = f * (st.sy + y * st.s);
    st.s *= f;
    st.m = m;
}

template <bool kEntropy>
__device__ __forceinline__ void add(Stats& st, float x, float ref, float c) {
    const float y = below(x, ref, c), e = __builtin_amdgcn_exp2f(y);
    st.s += e;
    if (kEntropy) st.sy += e * fmaxf(y, -1e30f);  // 0 * -inf: entries of no probability add nothing
}

// kCount vectors more.  kQuick: two operations an element less, of eleven, with y = x c - m c in one and without the
// guard of entropies; not finite, or nothing, where m c overflows or an entry is -inf, and not exact where m c is large
// (see quick_holds).  What the rounding of m c has moved all y by is put right in the sums.
template <typename T, bool kEntropy, bool kQuick, int kCount>
__device__ __forceinline__ void add_vecs(Stats& st, const vec_t* v, float c) {
    float m = st.m;
#pragma unroll
    for (int u = 0; u < kCount; ++u) {
        float f[kVec<T>];
        unpack<T>(v[u], f);
#pragma unroll
        for (int k = 0; k < kVec<T>; ++k) m = fmaxf(m, f[k]);
    }
    move_to<kEntropy>(st, m, c);
    const float ref = reference(m), shift = -ref * c;
    float s = 0.f, sy = 0.f;
#pragma unroll
    for (int u = 0; u < kCount; ++u) {
        float f[kVec<T>];
        unpack<T>(v[u], f);
#pragma unroll
        for (int k = 0; k < kVec<T>; ++k) {
            if constexpr (kQuick) {
                const float y = __builtin_fmaf(f[k], c, shift), e = __builtin_amdgcn_exp2f(y);
                s += e;
                if (kEntropy) sy = __builtin_fmaf(e, y, sy);
            } else {
                add<kEntropy>(st, f[k], ref, c);
            }
        }
    }
    if constexpr (kQuick) {
        const float off = __builtin_fmaf(-ref, c, -shift);  // below 2^-24 |m c|, and so small that 2^off is 1 + off ln 2
        s = __builtin_fmaf(s * off, kLn2, s);
        st.s += s;
        if (kEntropy) st.sy += __builtin_fmaf(s, off, __builtin_fmaf(sy * off, kLn2, sy));
    }
}

// Whether quick statistics of a row are the row's: its largest logit has put 1 into s, to within rounding, nothing
// overflowed, and the rounding of m c is at most 2^-13, so that what 1 + off ln 2 leaves out is below 2^-28 of s (at
// |m c| = 2^17 it would be 2^-18, at 2^24 a sixteenth).  A thread's own m c, below the row's, is either within twice the
// level as well or so far below that it has no part in s.
constexpr float kQuickLevel = 4096.f;
template <bool kEntropy>
__device__ __forceinline__ bool quick_holds(const Stats& st, float c) {
    return fabsf(st.m * c) <= kQuickLevel && st.s > 0.5f && st.s < INFINITY && (!kEntropy || fabsf(st.sy) < INFINITY);
}

// The statistics of vectors from + threadIdx.x, + kThreads_, ... below `to`; change(v, n) is applied to vector n.
template <typename T, bool kEntropy, bool kQuick, int kThreads_, bool kKeep = false, typename Change>
__device__ __forceinline__ void read_vecs(Stats& st, const void* vecs, int from, int to, float c, Change change) {
    // Two: more take the registers of waves that would hide the exponentials (8192 x 50257 bf16 with entropies: 93 us with
    // four, 87 with three, 84 with two, 91 with one).
    constexpr int kUnroll = 2;
    const int t = threadIdx.x;
    vec_t v[kUnroll];
    int n = from;
    for (; n + kUnroll * kThreads_ <= to; n += kUnroll * kThreads_) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) v[u] = load_vec<kKeep>(vecs, n + u * kThreads_, t);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) change(v[u], n + u * kThreads_ + t);
        add_vecs<T, kEntropy, kQuick, kUnroll>(st, v, c);
    }
    // what is left is on its way all at once, too
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const int first = n + u * kThreads_;
        v[u] = first + t < to ? load_vec<kKeep>(vecs, first, t) : nothing<T>();
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
        if (n + u * kThreads_ < to) {
            const bool in = n + u * kThreads_ + t < to;
            change(v[u], n + u * kThreads_ + t);
            if (!kQuick || in) add_vecs<T, kEntropy, kQuick, 1>(st, v + u, c);
        }
}

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) x = fmaxf(x, __shfl_xor(x, o, 64));
    return x;
}

template <bool kEntropy>
__device__ __forceinline__ Stats over_wave(Stats st, float c) {
    move_to<kEntropy>(st, wave_max(st.m), c);
    st.s = wave_sum(st.s);
    if (kEntropy) st.sy = wave_sum(st.sy);
    return st;
}

// The workgroup's statistics from its waves', through `lds` (one a wave).  One barrier, between writing and reading.
template <bool kEntropy, int kThreads_>
__device__ __forceinline__ Stats over_block(const Stats& wave, float c, Stats* lds) {
    constexpr int kN = kThreads_ / 64;
    Stats st = wave;
    if constexpr (kN > 1) {
        if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = wave;
        __syncthreads();
        st = lds[threadIdx.x % kN];
    }
    float m = st.m;
#pragma unroll
    for (int o = kN / 2; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    move_to<kEntropy>(st, m, c);
#pragma unroll
    for (int o = kN / 2; o >= 1; o >>= 1) {
        st.s += __shfl_xor(st.s, o, 64);
        if (kEntropy) st.sy += __shfl_xor(st.sy, o, 64);
    }
    return st;
}

// Loads come back in the order of their issue, and waiting for one is waiting for all before it: what a row needs beside
// its vectors is loaded before them, so that they are worked on as they arrive.
//
// A row in the registers of a workgroup: vector i kThreads + t of the row is v[i] of thread t, single element t its
// `single`.  Rows longer than that (kRest) have their remaining vectors read twice.
template <typename T, int kThreads_, int kVecs, bool kRest>
struct HeldRow {
    const T* row;
    Span span;
    vec_t v[kVecs];
    Raw<T> single_;
    static constexpr int kGroup = kVecs < 4 ? kVecs : 4, kGroups = kVecs / kGroup;
    // float: v holds 2^y below its group's, once the statistics are taken; -inf of a group of zeros, whatever the row's m
    float group_ref[kGroups];

    __device__ __forceinline__ const void* vecs() const { return row + span.head; }

    __device__ __forceinline__ bool has_single() const { return int(threadIdx.x) < span.extra; }
    __device__ __forceinline__ float single() const { return has_single() ? single_.value() : -INFINITY; }

    // `spare`: 16 bytes on their boundary that can be read, for rows without a vector.
    __device__ __forceinline__ void load(const T* row_, int vocab, const void* spare) {
        row = row_;
        span = span_of(row_, vocab);
        single_ = raw_at(row_ + (has_single() ? extra_element<T>(span, threadIdx.x) : 0));
        if constexpr (!kRest) load_held(spare);
    }

    // All kVecs loads whatever the row's length, the last vector again where there is none: with loads that are skipped
    // the compiler could not count how many are on their way, and would wait for all of them at the first.
    __device__ __forceinline__ void load_held(const void* spare) {
        const void* from = span.vecs > 0 ? vecs() : spare;
        const int last = max(span.vecs - 1, 0);
#pragma unroll
        for (int i = 0; i < kVecs; ++i) v[i] = load_vec(from, 0, min(i * kThreads_ + int(threadIdx.x), last));
    }

    // Vector i, where it is beyond the row, holds nothing.
    __device__ __forceinline__ void end_row(int i) {
        if ((i + 1) * kThreads_ > span.vecs && i * kThreads_ + int(threadIdx.x) >= span.vecs) v[i] = nothing<T>();
    }

    // fn(vector, its number less threadIdx.x) for each held one in turn.  The empty statement keeps the compiler from
    // unpacking all of them once and for both passes, which takes twice the registers.
    template <typename Fn>
    __device__ __forceinline__ void each(Fn fn) {
#pragma unroll
        for (int i = 0; i < kVecs; ++i)
            if (i * kThreads_ < span.vecs) {
                asm volatile("" : "+v"(v[i]));
                fn(v[i], i * kThreads_);
            }
    }

    // The thread's statistics.  hold(vector, i) is applied to held vector i, change(vector, number) to those that are not
    // held.  With kRest those held are loaded last, for the registers.
    template <typename Hold, typename Change>
    __device__ __forceinline__ Stats stats(float c, Hold hold, Change change) {
        Stats st = no_stats();
        if constexpr (kRest) {
            read_vecs<T, false, false, kThreads_, true>(st, vecs(), kVecs * kThreads_, span.vecs, c, change);
            load_held(row);  // never without a vector
        }
        // In groups, each as its loads arrive: the sum is taken below the thread's largest logit so far and moved when
        // that grows, so that only the reductions are left once the last load is there.
        move_to<false>(st, fmaxf(st.m, single()), c);
        add<false>(st, single(), reference(st.m), c);
#pragma unroll
        for (int q = 0; q < kGroups; ++q)
            if (q * kGroup * kThreads_ < span.vecs) {
                float m = st.m;
#pragma unroll
                for (int i = q * kGroup; i < (q + 1) * kGroup; ++i) {
                    end_row(i);
                    hold(v[i], i);
                    float f[kVec<T>];
                    unpack<T>(v[i], f);
#pragma unroll
                    for (int k = 0; k < kVec<T>; ++k) m = fmaxf(m, f[k]);
                }
                move_to<false>(st, m, c);
                group_ref[q] = m;
                const float ref = reference(m);
#pragma unroll
                for (int i = q * kGroup; i < (q + 1) * kGroup; ++i) {
                    asm volatile("" : "+v"(v[i]));
                    float f[kVec<T>];
                    unpack<T>(v[i], f);
#pragma unroll
                    for (int k = 0; k < kVec<T>; ++k) {
                        f[k] = __builtin_amdgcn_exp2f(below(f[k], ref, c));
                        st.s += f[k];
                    }
                    if constexpr (sizeof(T) == 4) v[i] = pack<T>(f);
                }
                __builtin_amdgcn_sched_barrier(0);  // the next group is not begun, and waited for, before
            }
        return st;
    }

    // g_j = b 2^y below m.
    template <typename Change>
    __device__ __forceinline__ void write(T* __restrict__ g, float b, float m, float c, Change change) {
        T* at = g + span.head;
        const int t = threadIdx.x;
        each([&](vec_t& x, int n) {
            float f[kVec<T>];
            unpack<T>(x, f);
            const float group =
                sizeof(T) == 4 ? b * __builtin_amdgcn_exp2f(below(group_ref[n / kThreads_ / kGroup], m, c)) : b;
#pragma unroll
            for (int k = 0; k < kVec<T>; ++k)
                f[k] = group * (sizeof(T) == 4 ? f[k] : __builtin_amdgcn_exp2f(below(f[k], m, c)));
            if (n + t < span.vecs) store_vec(at, n, t, pack<T>(f));
        });
        if constexpr (kRest) {
            constexpr int kUnroll = 4;
            for (int n = kVecs * kThreads_; n < span.vecs; n += kUnroll * kThreads_) {
                vec_t x[kUnroll];
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) {
                    const int first = n + u * kThreads_;
                    x[u] = first + t < span.vecs ? load_vec(vecs(), first, t) : nothing<T>();
                }
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) {
                    const int first = n + u * kThreads_;
                    change(x[u], first + t);
                    float f[kVec<T>];
                    unpack<T>(x[u], f);
#pragma unroll
                    for (int k = 0; k < kVec<T>; ++k) f[k] = b * __builtin_amdgcn_exp2f(below(f[k], m, c));
                    if (first + t < span.vecs) store_vec(at, first, t, pack<T>(f));
                }
            }
        }
        if (has_single())
            g[extra_element<T>(span, threadIdx.x)] = narrow<T>(b * __builtin_amdgcn_exp2f(below(single(), m, c)));
    }
};

struct Unchanged {
    __device__ __forceinline__ void operator()(vec_t&, int) const {}
};

// The number that weights are divided by: rows that count, or sequences that have any.  Every wave by itself; the load
// of the first 64 counts is apart, to be on its way before a row's.
struct Counts {
    const int32_t* count;
    int64_t items;
    int32_t first;

    __device__ __forceinline__ Counts(const int32_t* count_, int64_t items_)
        : count(count_), items(items_),
          first(count_[max(min(int64_t(threadIdx.x % 64), items_ - 1), int64_t(0))]) {}
    __device__ __forceinline__ float all() const {
        const int lane = threadIdx.x % 64;
        float n = lane < items ? float(first) : 0.f;
        for (int64_t i = 64 + lane; i < items; i += 64) n += float(count[i]);
        return fmaxf(wave_sum(n), 1.f);
    }
};

// ---- the sum over all rows

// Where a launch's workgroups leave their parts of the result.  With a ticket (0 before the launch) the last of them adds
// up all of them, in the order of their numbers; without one a launch of result_kernel does.
struct Result {
    float4* parts;     // NULL: the result is not asked for
    uint32_t* ticket;
    uint32_t of;       // workgroups
    float* result;     // f times the sum of x, the sums of y and z
    float f;
};

// By all of a workgroup's threads, at its end.
__device__ __forceinline__ void put_part(const Result& out, uint32_t i, float x, float y, float z) {
    if (!out.parts || threadIdx.x >= 64) return;
    if (!out.ticket) {
        if (threadIdx.x == 0) out.parts[i] = make_float4(x, y, z, 0.f);
        return;
    }
    uint32_t before = 0;
    if (threadIdx.x == 0) {
        float* part = reinterpret_cast<float*>(out.parts + i);
        __hip_atomic_store(part, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(part + 1, y, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(part + 2, z, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        before = __hip_atomic_fetch_add(out.ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (uint32_t(__builtin_amdgcn_readfirstlane(int(before))) != out.of - 1) return;
    float sum[3] = {0.f, 0.f, 0.f};
    for (uint32_t k = threadIdx.x; k < out.of; k += 64) {
        const float* part = reinterpret_cast<const float*>(out.parts + k);
#pragma unroll
        for (int j = 0; j < 3; ++j) sum[j] += __hip_atomic_load(part + j, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
#pragma unroll
    for (int j = 0; j < 3; ++j) sum[j] = wave_sum(sum[j]);
    if (threadIdx.x == 0) {
        out.result[0] = sum[0] * out.f;
        out.result[1] = sum[1];
        out.result[2] = sum[2];
    }
}

// ---- launches

// Waves that should fit a SIMD beside each other: 512 registers shared among them, kVecs * 4 a wave for the row and
// some 40 to 60 for the rest.
template <int kVecs>
constexpr int kRowWaves = kVecs > 8 ? 4 : kVecs > 4 ? 5 : kVecs > 2 ? 6 : 8;

inline Rows make_rows(const mamw_rows& x, float temperature) {
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

inline PerRow make_per_row(const mamw_per_row& a) {
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

inline double row_bytes(const mamw_rows& x, bool grad) {
    return double(x.outer * x.inner) * double(x.vocab) * (x.type == MAMW_F32 ? 4.0 : 2.0) * (grad ? 2.0 : 1.0);
}

// fn(workgroup size, vectors a thread, whether some are left) for rows of `vecs` vectors, held by one workgroup.  Four
// vectors a thread, as long as there are threads for it, measured best; halves and doubles of it, us for 1.6 GB:
//     4000 bf16 (500 vectors)     128 x 4: 151   256 x 2: 158   512 x 1: 271
//     8000 (1000)                 128 x 8: 167   256 x 4: 159   512 x 2: 175
//     16000 (2000)                256 x 8: 161   512 x 4: 152  1024 x 2: 181
//     32000 (4000)               256 x 16: 157   512 x 8: 155  1024 x 4: 145
//     50257 (6282)               512 x 16: 248  1024 x 8: 244
// That is for a kernel of few registers: two workgroups of 1024 share a compute unit if a thread takes 64 at most.  One
// of more has workgroups of 512 for the long rows (distillation with a rest: 32000 bf16 152 with 512 x 8, 159 with
// 1024 x 4; 50257 266 with 512 x 16, 322 with 1024 x 8).
// A row of 256 KiB is all the registers of a compute unit that its other values leave.  A longer row keeps that much and
// has the rest read twice.
template <int kN>
struct Int {
    static constexpr int value = kN;
};
template <bool kMoreRegisters, typename Fn>
int with_held_row(int64_t vecs, Fn fn) {
    if (vecs <= 256) return fn(Int<128>(), Int<2>(), Int<0>());
    if (vecs <= 512) return fn(Int<128>(), Int<4>(), Int<0>());
    if (vecs <= 1024) return fn(Int<256>(), Int<4>(), Int<0>());
    if (vecs <= 2048) return fn(Int<512>(), Int<4>(), Int<0>());
    if constexpr (kMoreRegisters) {
        if (vecs <= 4096) return fn(Int<512>(), Int<8>(), Int<0>());
        if (vecs <= 8192) return fn(Int<512>(), Int<16>(), Int<0>());
    } else {
        if (vecs <= 4096) return fn(Int<1024>(), Int<4>(), Int<0>());
        if (vecs <= 8192) return fn(Int<1024>(), Int<8>(), Int<0>());
    }
    if (vecs <= 16384) return fn(Int<1024>(), Int<16>(), Int<0>());
    return fn(Int<1024>(), Int<16>(), Int<1>());
}

// One workgroup a row.  Such workgroups come and go by themselves: a row's loads do not wait for the stores of the row
// before, as they would in a loop over rows, where the same counter covers both (65536 x 4096 bf16: 205 us in 2048
// workgroups, 180 in 65536).
inline dim3 row_grid(int64_t rows) {
    const unsigned most = 1u << 16;
    return rows <= int64_t(most) ? dim3(unsigned(rows)) : dim3(most, unsigned((rows + most - 1) / most));
}

// Up to this many workgroups the last one adds up the result, above a kernel of its own does.  The launch saved is 4 us on
// the device and as many on the host; the ticket costs each workgroup a write-back of its L2 cache (64 rows: 6 us
// instead of 5 and 4 for the other launch; 256 x 50257 fp32: 30 instead of 18 and 4; 1024: 124 instead of 67 and 4).
constexpr int64_t kTickets = 64;

// Where the rows' parts of `result` go; `launched`: the ticket is cleared by a launch before.
inline Result make_result(const ObjectiveWorkspace& ws, char* base, int64_t rows, bool launched, float f, float* result) {
    Result out;
    out.parts = reinterpret_cast<float4*>(base + ws.partials_at);
    out.ticket = launched && rows <= kTickets ? reinterpret_cast<uint32_t*>(base + ws.ticket_at) : nullptr;
    out.of = uint32_t(rows);
    out.result = result;
    out.f = f;
    return out;
}

// Defined in objectives.hip.
int launch_count(const Rows& rows, const PerRow& tokens, int64_t ignore, const PerRow& mask, const Sequences& seqs,
                 const ObjectiveWorkspace& ws, bool by_sequence, char* base, hipStream_t stream);
// result_kernel, where the workgroups had no ticket.
int launch_result(const Result& out, const ObjectiveWorkspace& ws, char* base, hipStream_t stream);

}  // namespace mamw
