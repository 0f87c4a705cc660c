// Distillation from a teacher's top logits for MI355X (gfx950): the selection of the top logits, and the loss of a
// student's logits against them with its gradient.
//
// With z a row of the student's logits, t_i the teacher's values at the indices j_i, tau the temperature, w the weight:
//   p_i = exp(t_i / tau - Lt)                     Lt = logsumexp(t / tau [, rest])
//   q_j = exp(z_j / tau - L)                      L = logsumexp(z / tau),  q_rest = the sum of q outside the top set
//   KL = sum p_i (log p_i - log q_{j_i}) [+ p_rest (log p_rest - log q_rest)]
//   loss = mean of w tau^2 KL + (1 - w) (logsumexp(z) - z_target)
//   dz_j = g / n (w tau (q_j f_j - p_j) + (1 - w) (s_j - [j = target])),  s = softmax(z),
//   f_j = 1 - p_rest / q_rest outside the top set where rest is a class, else 1 (p_j = 0 outside the top set).
//
// A student near its teacher has a loss far below L, so the loss is a small difference of terms that share L. The sum over
// the row, in fp32, therefore leaves out the top set and the target (a bitmap in LDS marks them); their terms, and all that
// is joined from them, are computed in fp64, where the shared part cancels. An error of the row's sum then reaches KL only
// times (q_rest - p_rest).
//
// All of it is bound by HBM: the forward reads the logits once, the backward reads them once and writes the gradient.
// Built with NaN semantics: NaN and infinite logits reach the outputs.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

#include "nanonemo_distill.h"
#include "rows.h"

#define NNDIS_API extern "C" __attribute__((visibility("default")))

namespace {

constexpr int kMaxTop = 512;
constexpr int kMaxVocab = 393216;  // 48 KB of marks
constexpr int kVocabBits = 19;
constexpr long long kIgnore = -100;
constexpr float kL2e = 1.4426950408889634f;

struct Layout {  // row r at (r / T) * sb + (r % T) * st
    long long sb, st;
    int T;
    __device__ long long at(int r) const {
        const int b = r / T;
        return b * sb + (r - b * T) * st;
    }
};

// A 16-byte group at an address of the element's own alignment.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
template <int DT>
__device__ inline u32x4 load_any(const typename Row<DT>::T* p) {
    return *reinterpret_cast<const u32x4_any*>(p);
}
// (Past the caches, which keep what else the step needs: the gradient is as large as the logits. 8192 x 50304 bf16: the backward
// 321 us with cached stores, 297 so, and the next forward 160 and 142.)
template <int DT>
__device__ inline void store_any(typename Row<DT>::T* p, u32x4 v) {
    __builtin_nontemporal_store((u32x4_any)v, reinterpret_cast<u32x4_any*>(p));
}
template <int DT>
__device__ inline typename Row<DT>::T minus_inf() {
    if constexpr (DT == kF32)
        return -INFINITY;
    else
        return DT == kBF16 ? 0xff80 : 0xfc00;
}
// Group i of a row; values past the row's end are -inf.
template <int DT>
__device__ inline u32x4 group(const typename Row<DT>::T* row, int i, int V) {
    using R = Row<DT>;
    const int j = i * R::W;
    if (j + R::W <= V) return load_any<DT>(row + j);
    union {
        u32x4 v;
        typename R::T e[R::W];
    } u;
#pragma unroll
    for (int e = 0; e < R::W; ++e) u.e[e] = j + e < V ? row[j + e] : minus_inf<DT>();
    return u.v;
}

// Group i of a row of at least W values, from min(i W, V - W) on: the last one of a row that is not whole groups overlaps the
// one before. Then own() makes what the group before holds (all of a group past the row's end) -inf: apart, so that many loads
// can be under way.
template <int DT>
__device__ inline u32x4 group_at(const typename Row<DT>::T* row, int i, int V) {
    constexpr int W = Row<DT>::W;
    const uint32_t bytes = (uint32_t)min(i * W, V - W) * (uint32_t)sizeof(typename Row<DT>::T);  // (32 bits: the row's address stays scalar)
    return load_any<DT>(reinterpret_cast<const typename Row<DT>::T*>(reinterpret_cast<const char*>(row) + bytes));
}
template <int DT>
__device__ inline void own(u32x4& v, int i, int V) {
    constexpr int W = Row<DT>::W;
    const int twice = i * W - (V - W);
    if (twice <= 0) return;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if constexpr (DT == kF32) {
            if (w < twice) v[w] = 0xff800000u;
        } else {
            constexpr uint32_t ninf = DT == kBF16 ? 0xff80u : 0xfc00u;
            if (2 * w < twice) v[w] = (v[w] & 0xffff0000u) | ninf;
            if (2 * w + 1 < twice) v[w] = (v[w] & 0xffffu) | (ninf << 16);
        }
    }
}

// Sums, maxima and the like over a block of TB threads: every thread gets the result. `tmp` is one value per wave, free for
// the next call as soon as this one has returned everywhere.
template <int TB, typename T, typename F>
__device__ inline T block_all(T v, T* tmp, F f) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v = f(v, __shfl_xor(v, d));
    if constexpr (TB > 64) {
        if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = v;
        __syncthreads();
        v = tmp[0];
#pragma unroll
        for (int w = 1; w < TB / 64; ++w) v = f(v, tmp[w]);
        __syncthreads();
    }
    return v;
}

// ------------------------------------------------------------------------------------------
// Softmax sums.
// ------------------------------------------------------------------------------------------
// exp((x - m) * c / log2(e)), the difference rounded first; 0 for x = -inf whatever a finite m.
__device__ inline float exp_diff(float x, float m, float c) { return __builtin_amdgcn_exp2f((x - m) * c); }
// What exponents are relative to: 0 where every value is -inf (their exp is 0 then) or one is +inf (infinite then).
__device__ inline float base_of(float m) { return fabsf(m) == INFINITY ? 0.f : m; }

// Whether a sum of exponentials relative to a value of the caller's choice can stand: those below 2^-126 count as 0, of up to
// kMaxVocab of them 5e-33 in all, which has to be nothing beside the sum (5e-8 at 1e-25; of 1e-30 it was 0.5 %).
__device__ inline bool stands(float s) { return s > 1e-25f && s < 1e30f; }

// The factor that takes a sum relative to base_of(m) to another base; 0 for the empty sum, whose m is -inf.
__device__ inline float rebase(float m, float base, float c) { return exp_diff(m == INFINITY ? 0.f : m, base, c); }

struct MaxSum {  // s = sum of exp((x - base_of(m)) / tau); with a second sum at temperature 1
    float m, s, s1;
};
template <bool BOTH>
__device__ inline MaxSum merge(MaxSum a, MaxSum b, float c) {
    const float m = fmaxf(a.m, b.m), base = base_of(m);
    MaxSum r{m, a.s * rebase(a.m, base, c) + b.s * rebase(b.m, base, c), 0.f};
    if constexpr (BOTH) r.s1 = a.s1 * rebase(a.m, base, kL2e) + b.s1 * rebase(b.m, base, kL2e);
    return r;
}
// W further values.
template <bool BOTH, int W>
__device__ inline void take(MaxSum& a, const float* v, float c) {
    float m = a.m;
#pragma unroll
    for (int e = 0; e < W; ++e) m = fmaxf(m, v[e]);
    const float base = base_of(m);
    float s = a.s * rebase(a.m, base, c), s1 = BOTH ? a.s1 * rebase(a.m, base, kL2e) : 0.f;
#pragma unroll
    for (int e = 0; e < W; ++e) {
        s += exp_diff(v[e], base, c);
        if constexpr (BOTH) s1 += exp_diff(v[e], base, kL2e);
    }
    a = {m, s, s1};
}
template <int TB, bool BOTH>
__device__ inline MaxSum block_merge(MaxSum a, MaxSum* tmp, float c) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1)
        a = merge<BOTH>(a, MaxSum{__shfl_xor(a.m, d), __shfl_xor(a.s, d), BOTH ? __shfl_xor(a.s1, d) : 0.f}, c);
    if constexpr (TB > 64) {
        if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = a;
        __syncthreads();
        a = tmp[0];
#pragma unroll
        for (int w = 1; w < TB / 64; ++w) a = merge<BOTH>(a, tmp[w], c);
        __syncthreads();
    }
    return a;
}

// ------------------------------------------------------------------------------------------
// The top logits: one block per row.
// ------------------------------------------------------------------------------------------
// A logit as a whole number of the same order: -0 as 0, NaN above everything; 0 is below every logit.
template <int DT>
struct Key {
    static constexpr int kBits = DT == kF32 ? 32 : 16;
    static constexpr uint32_t kSign = 1u << (kBits - 1), kAll = DT == kF32 ? 0xffffffffu : 0xffffu;
    static constexpr uint32_t kInf = DT == kF32 ? 0x7f800000u : DT == kBF16 ? 0x7f80u : 0x7c00u;
    using T = typename Row<DT>::T;
    static __device__ uint32_t of(T x) {
        uint32_t u;
        if constexpr (DT == kF32)
            u = __float_as_uint(x);
        else
            u = x;
        const uint32_t mag = u & (kSign - 1);
        if (mag > kInf) return kAll;
        if (mag == 0) u = 0;
        return u & kSign ? u ^ kAll : u | kSign;
    }
    static __device__ T value(uint32_t key) {
        const uint32_t u = key & kSign ? key ^ kSign : key ^ kAll;
        if constexpr (DT == kF32)
            return __uint_as_float(u);
        else
            return (T)u;
    }
};
// A key and the place of its value as one number: the larger key first, of equal ones the lower place. A double holds the 51
// bits exactly, and two of them are compared in one instruction of full rate (two 64-bit integers take four times as long).
__device__ inline double ranked(uint32_t key, int j) { return fma((double)key, (double)(1 << kVocabBits), (double)((1 << kVocabBits) - 1 - j)); }
__device__ inline uint32_t key_in(double r) { return (uint32_t)(r * (1.0 / (1 << kVocabBits))); }
__device__ inline int place_in(double r) { return (1 << kVocabBits) - 1 - (int)(r - (double)key_in(r) * (double)(1 << kVocabBits)); }

// Largest values as whole numbers, for a group of 16 bytes at a time: like Key, but -0 below 0 and a NaN by its sign (the largest
// value shows one without it; one with it makes the sum of exponentials NaN).
template <int DT>
struct Order {
    using K = Key<DT>;
    static __device__ uint32_t of(uint32_t u) { return u & K::kSign ? u ^ K::kAll : u | K::kSign; }
    static __device__ typename K::T value(uint32_t order) { return K::value(order); }  // (the same for both orders)
    static constexpr uint32_t kZero = K::kSign, kMinusZero = kZero - 1, kMinusInf = K::kAll ^ (K::kSign | K::kInf), kPlusInf = K::kSign | K::kInf;
    // As signed whole numbers, values that are not negative have the order of floats and negative ones its reverse: the largest
    // value is the largest of them, or the least where all are negative.
    static __device__ uint32_t most(u32x4 raw) {
        int hi, lo;
        if constexpr (DT == kF32) {
            hi = max(max((int)raw[0], (int)raw[1]), max((int)raw[2], (int)raw[3]));
            lo = min(min((int)raw[0], (int)raw[1]), min((int)raw[2], (int)raw[3]));
        } else {
            typedef short s16x2 __attribute__((ext_vector_type(2)));
            s16x2 x[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) x[w] = __builtin_bit_cast(s16x2, (uint32_t)raw[w]);
            const s16x2 h = __builtin_elementwise_max(__builtin_elementwise_max(x[0], x[1]), __builtin_elementwise_max(x[2], x[3]));
            const s16x2 l = __builtin_elementwise_min(__builtin_elementwise_min(x[0], x[1]), __builtin_elementwise_min(x[2], x[3]));
            hi = max((int)h[0], (int)h[1]), lo = min((int)l[0], (int)l[1]);
        }
        return of((uint32_t)(hi >= 0 ? hi : lo) & K::kAll);
    }
};

// A bound that at least k of a wave's 64 P values reach, and at most k / 16 + 2 more where equal values allow it, found bit by
// bit.
template <int BITS, int P>
__device__ inline uint32_t reached(const uint32_t (&v)[P], int k) {
    uint32_t found = 0;
    for (int b = BITS - 1; b >= 0; --b) {
        const uint32_t t = found | (1u << b);
        int reach = 0;
#pragma unroll
        for (int i = 0; i < P; ++i) reach += __popcll(__ballot(v[i] >= t));
        if (reach < k) continue;
        found = t;
        if (reach <= k + k / 16 + 2) break;
    }
    return found;
}

// What a row's selection keeps in LDS.
template <int TB>
struct TopShared {
    static constexpr int kWaves = TB / 64;
    static constexpr int kCandidates = TB == 64 ? 640 : 1024;  // (at least kMaxTop)
    static constexpr int kList = TB == 64 ? 1 : TB == 256 ? 64 : 1024 / kWaves;  // groups of a wave's list
    double cand[kCandidates];  // (ranked)
    u32x4 list[kWaves][kList];
    int list_at[kWaves][kList];
    float below[TB == 64 ? 1 : kCandidates];  // exponentials of the candidates that are not among the k
    uint32_t bins[TB == 64 ? 1 : 1024];
    int tmp[kWaves];
    float tmpf[kWaves];
    MaxSum sums[kWaves];
    int count, special, full;
    uint32_t bound;
    double last;
};

// One block of TB threads per row. A thread holds NV groups of the row in registers from its one load to the end (the row is
// read once); NV = 0 is for rows too long for that, which are read twice.
//
//   1  The k-th largest of some hundred parts' largest values is a bound that at least k values reach, and few more do.
//   2  Values that reach it are the candidates (their groups go to a list of the wave's, so that the code for single values is
//      there once); the exponentials of all others are summed.
//   3  A candidate's rank is the number of larger ones; those behind the k join the sum.
//
// Measured at 8192 x 50304 bf16, k = 64: 161 us (5.1 TB/s), three rows to a CU at 80 registers, where a row's search and
// ranking hide behind the others' loads. With the row read again for every step it took 700 us, with 1024 threads of 64
// registers (7 groups each, 27 of them spilled) 390, and 180 where a part's largest value took four instructions a pair of
// values and NaN another two. A single row takes 10 us, most of it the steps' latency.
// Rows for which the above does not do (many equal values, NaN, more candidates than the lists hold: with 256 threads from a k of
// about 150 on, 8192 x 8192 bf16 takes 76 us at k = 128 and 1005 at 256) take a search of the k-th value bit by bit instead, and
// rows whose others lie far below the bound a sum relative to their own largest.
template <int DT, int TB, int NV>
__global__ __launch_bounds__(TB, TB == 512 && NV <= 13 ? 6 : 4) void top_kernel(const void* __restrict__ logits, Layout at, void* __restrict__ values,
                                                    long long* __restrict__ indices, float* __restrict__ rest, int V, int k, float c,
                                                    double inv_tau) {
    using R = Row<DT>;
    using T = typename R::T;
    using K = Key<DT>;
    using O = Order<DT>;
    using S = TopShared<TB>;
    constexpr int N = NV ? NV : 1;
    const T* row = reinterpret_cast<const T*>(logits) + at.at(blockIdx.x);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, groups = (V + R::W - 1) / R::W;
    __shared__ S sh;
    union Group {
        u32x4 v;
        T e[R::W];
    };
    u32x4 raw[N];
    uint32_t most[N];  // the order of each group's largest value
    auto bits_of = [](T x) {
        if constexpr (DT == kF32)
            return __float_as_uint(x);
        else
            return (uint32_t)x;
    };
    auto begin_of = [&](int i) { return V < R::W ? 0 : min(i * R::W, V - R::W); };
    auto one_group = [&](int i) {
        u32x4 v = group_at<DT>(row, i, V);
        own<DT>(v, i, V);
        return v;
    };
    auto each = [&](auto f) {  // (the row again, for the steps that few rows take)
        for (int i = tid; i < groups; i += TB) {
            Group u;
            u.v = group<DT>(row, i, V);
#pragma unroll
            for (int e = 0; e < R::W; ++e)
                if (i * R::W + e < V) f(u.e[e], i * R::W + e);
        }
    };
    auto add = [](auto a, auto b) { return a + b; };
    if (tid == 0) sh.count = 0, sh.special = 0, sh.full = 0;
    __syncthreads();

    // 1. The parts: four threads' values, a thread's, a group's, or (one wave) every value. Of 256 parts, 64 leave 74
    // candidates; of 1024, 512 leave 710.
    uint32_t mine = 0, least = 0;
    if constexpr (NV > 0) {
#pragma unroll
        for (int n = 0; n < NV; ++n) raw[n] = TB == 64 && V < R::W ? group<DT>(row, 0, tid + n ? 0 : V) : group_at<DT>(row, tid + n * TB, V);
        if (TB > 64 || V >= R::W) {
#pragma unroll
            for (int n = 0; n < NV; ++n) own<DT>(raw[n], tid + n * TB, V);
        }
#pragma unroll
        for (int n = 0; n < NV; ++n) mine = max(mine, most[n] = O::most(raw[n]));
    } else {
        for (int i = tid; i < groups; i += TB) mine = max(mine, O::most(one_group(i)));
    }
    if constexpr (TB == 64) {
        if (2 * k <= groups) {
            least = reached<K::kBits>(most, k);
        } else {
            uint32_t v[N * R::W];
#pragma unroll
            for (int n = 0; n < N; ++n) {
                Group u;
                u.v = raw[n];
#pragma unroll
                for (int e = 0; e < R::W; ++e) v[n * R::W + e] = O::of(bits_of(u.e[e]));
            }
            least = reached<K::kBits>(v, k);
        }
        if (__ballot(mine > O::kPlusInf)) least = 0;
        if (least == O::kZero) least = O::kMinusZero;  // (they are equal)
    } else {
        if (mine > O::kPlusInf) sh.special = 1;
        int parts = 0;
        if (4 * k <= TB / 4) {
            mine = max(mine, (uint32_t)__shfl_xor((int)mine, 1));
            mine = max(mine, (uint32_t)__shfl_xor((int)mine, 2));
            parts = TB / 4;
            if (tid % 4 == 0) sh.bins[tid / 4] = mine;
        } else if (NV > 0 ? 4 * k <= TB : 2 * k <= TB) {
            parts = TB;
            sh.bins[tid] = mine;
        } else if (NV > 0 && k <= groups) {
            parts = min(NV * TB, 1024);
            // (of more groups than parts, several make one)
#pragma unroll
            for (int n = 0; n < N; ++n)
                if (n * TB + tid < 1024) {
                    uint32_t m = most[n];
#pragma unroll
                    for (int o = n + 1024 / TB; o < N; o += 1024 / TB) m = max(m, most[o]);
                    sh.bins[n * TB + tid] = m;
                }
        }
        __syncthreads();
        if (tid < 64) {
            auto search = [&](auto p) {
                constexpr int P = decltype(p)::value;
                uint32_t v[P];
#pragma unroll
                for (int i = 0; i < P; ++i) v[i] = sh.bins[64 * i + tid];
                return reached<K::kBits>(v, k);
            };
            switch (parts / 64) {
                case 0: break;
                case 1: least = search(std::integral_constant<int, 1>()); break;
                case 2: least = search(std::integral_constant<int, 2>()); break;
                case 4: least = search(std::integral_constant<int, 4>()); break;
                case 8: least = search(std::integral_constant<int, 8>()); break;
                default: least = search(std::integral_constant<int, 16>());  // 1024
            }
            if (tid == 0) sh.bound = sh.special ? 0 : least == O::kZero ? O::kMinusZero : least;
        }
        __syncthreads();
        least = sh.bound;
    }

    // 2. Exponents are in powers of two relative to 2^b, the whole number b next to the bound's own exponent (so that x c - b is
    // rounded once).
    const float v_b = R::one(O::value(least)), b = rintf(v_b * c);
    float s = 0.f;
    auto e_of = [&](T x) { return __builtin_amdgcn_exp2f(fmaf(R::one(x), c, -b)); };
    bool quick = least > O::kMinusInf;  // (what lies past the row's end is -inf)
    int n = 0;
    if (quick) {
        if constexpr (TB == 64) {
#pragma unroll
            for (int m = 0; m < N; ++m) {
                Group u;
                u.v = raw[m];
#pragma unroll
                for (int e = 0; e < R::W; ++e) {
                    const bool hit = O::of(bits_of(u.e[e])) >= least;
                    const uint64_t hits = __ballot(hit);
                    s += hit ? 0.f : e_of(u.e[e]);
                    if (hits) {
                        const int to = n + __popcll(hits & ((1ull << lane) - 1));
                        if (hit && to < S::kCandidates) sh.cand[to] = ranked(K::of(u.e[e]), begin_of(tid + m * TB) + e);
                        n += __popcll(hits);
                    }
                }
            }
            if (__ballot(s != s)) n = S::kCandidates + 1;  // (a NaN)
            __syncthreads();
        } else {
            int on_list = 0;
            auto sweep = [&](u32x4 v, uint32_t m, int i) {
                const uint64_t hits = __ballot(m >= least);
                if (m >= least) {
                    const int to = on_list + __popcll(hits & ((1ull << lane) - 1));
                    if (to < S::kList) {
                        sh.list[wave][to] = v;
                        sh.list_at[wave][to] = i;
                    }
                } else {
                    float f[R::W];
                    R::widen(v, f);
#pragma unroll
                    for (int e = 0; e < R::W; ++e) s += __builtin_amdgcn_exp2f(fmaf(f[e], c, -b));
                }
                on_list += __popcll(hits);
            };
            if constexpr (NV > 0) {
#pragma unroll
                for (int m = 0; m < NV; ++m) sweep(raw[m], most[m], tid + m * TB);
            } else {
                for (int i = tid; i < groups; i += TB) {
                    const u32x4 v = one_group(i);
                    sweep(v, O::most(v), i);
                }
            }
            on_list = __builtin_amdgcn_readfirstlane(on_list);  // (the first lane has seen every group of the wave)
            if (on_list > S::kList) {
                if (lane == 0) sh.full = 1;
                on_list = S::kList;
            }
            if (s != s) sh.full = 1;  // (a NaN)
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (the wave's own list: no other's is read)
            __builtin_amdgcn_wave_barrier();
            for (int t = lane; t < on_list * R::W; t += 64) {
                const int g = t / R::W;
                const T x = reinterpret_cast<const T*>(sh.list[wave])[t];
                if (O::of(bits_of(x)) >= least) {
                    const int p = atomicAdd(&sh.count, 1);
                    if (p < S::kCandidates) sh.cand[p] = ranked(K::of(x), begin_of(sh.list_at[wave][g]) + t % R::W);
                } else {
                    s += e_of(x);
                    if (s != s) sh.full = 1;
                }
            }
            __syncthreads();
            n = sh.full ? S::kCandidates + 1 : sh.count;
        }
        quick = n <= S::kCandidates;
    }
    if (!quick) {
        // The k-th largest key, and the place of the last of its equals that belongs to the k.
        auto counted = [&](auto f) {
            int n = 0;
            each([&](T x, int j) { n += f(K::of(x), j) ? 1 : 0; });
            return block_all<TB>(n, sh.tmp, add);
        };
        uint32_t key_k = 0;
        for (int b = K::kBits - 1; b >= 0; --b) {
            const uint32_t t = key_k | (1u << b);
            if (counted([&](uint32_t key, int) { return key >= t; }) >= k) key_k = t;
        }
        const int need = k - counted([&](uint32_t key, int) { return key > key_k; });
        int place = 0;
        for (int b = kVocabBits - 1; b >= 0; --b) {
            const int t = place | (1 << b);
            if (counted([&](uint32_t key, int j) { return key == key_k && j < t; }) < need) place = t;
        }
        __syncthreads();
        if (tid == 0) sh.count = 0;
        __syncthreads();
        each([&](T x, int j) {
            const uint32_t key = K::of(x);
            if (key > key_k || (key == key_k && j <= place)) sh.cand[atomicAdd(&sh.count, 1)] = ranked(key, j);
        });
        __syncthreads();
        n = k;
    }
    // 3. Every wave holds all candidates, and ranks every kWaves-th one: a comparison with all of them is one instruction a 64, and
    // a count of its result bits.
    auto rank_all = [&](auto parts) {
        constexpr int P = decltype(parts)::value;
        double x[P];
#pragma unroll
        for (int i = 0; i < P; ++i) x[i] = 64 * i + lane < n ? sh.cand[64 * i + lane] : -1.0;
        for (int from = wave; from < n; from += 64 * S::kWaves) {  // 64 of the wave's, one for each lane in the end
            const int own = min(64, (n - from + S::kWaves - 1) / S::kWaves);
            const double my = lane < own ? sh.cand[from + lane * S::kWaves] : 0.0;
            const int lo = (int)__builtin_bit_cast(uint64_t, my), hi = (int)(__builtin_bit_cast(uint64_t, my) >> 32);
            int rank = 0;
            for (int t = 0; t < own; ++t) {
                const double y = __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane(lo, t) | (uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, t) << 32);
                int larger = 0;
#pragma unroll
                for (int i = 0; i < P; ++i) larger += __popcll(__ballot(x[i] > y));
                rank = lane == t ? larger : rank;
            }
            if (lane >= own) continue;
            const T v = K::value(key_in(my));
            if (rank >= k) {  // (one wave's candidates have one order; of several waves, they are summed by rank)
                if constexpr (TB == 64)
                    s += e_of(v);
                else
                    sh.below[rank - k] = e_of(v);
                continue;
            }
            const size_t to = (size_t)blockIdx.x * k + rank;
            reinterpret_cast<T*>(values)[to] = v;
            indices[to] = place_in(my);
            if (rank == k - 1) sh.last = my;
        }
    };
    switch ((n + 63) / 64) {
        case 1: rank_all(std::integral_constant<int, 1>()); break;
        case 2: rank_all(std::integral_constant<int, 2>()); break;
        case 3: rank_all(std::integral_constant<int, 3>()); break;
        case 4: rank_all(std::integral_constant<int, 4>()); break;
        case 5: case 6: rank_all(std::integral_constant<int, 6>()); break;
        case 7: case 8: rank_all(std::integral_constant<int, 8>()); break;
        default: rank_all(std::integral_constant<int, S::kCandidates / 64>());
    }
    __syncthreads();
    if (quick) {
        if constexpr (TB > 64)
            for (int i = tid; i < n - k; i += TB) s += sh.below[i];
        s = block_all<TB>(s, sh.tmpf, add);
        if (stands(s)) {
            // (c is log2(e) / tau rounded: what that puts on the exponents near the bound comes off again)
            const double ln2 = 0.6931471805599453, off = v_b * (inv_tau / ln2 - (double)c);
            if (tid == 0) rest[blockIdx.x] = (float)(ln2 * ((double)b + off + log2((double)s)));
            return;
        }
    }
    const double end = sh.last;
    MaxSum a{-INFINITY, 0.f, 0.f};
    each([&](T x, int j) {
        if (ranked(K::of(x), j) >= end) return;
        const float v = R::one(x);
        take<false, 1>(a, &v, c);
    });
    a = block_merge<TB, false>(a, sh.sums, c);
    if (tid == 0) rest[blockIdx.x] = (float)(base_of(a.m) * inv_tau + log((double)a.s));
}

// ------------------------------------------------------------------------------------------
// The loss: one block per row.
// ------------------------------------------------------------------------------------------
struct Loss {
    const void* logits;
    Layout at;
    const void* values;
    const long long* indices;
    const float* rest;         // or nullptr
    const long long* targets;  // or nullptr
    double* stats;             // [R][kStats], then the rows' losses [R], then 1 / n
    int V, k, vdt;
    float c;  // log2(e) / tau
    double tau, weight;
    __device__ bool hard() const { return targets && weight < 1.0; }
};
// A row's statistics: L, logsumexp(z), Lt, log of the rest's sum and p_rest, a logit that the gradient's exponents are relative to,
// and whether an index is there twice.
enum { kL, kL1, kLt, kLr, kPr, kBase, kTwice, kStats };

__device__ inline float value_at(const void* p, long long i, int dt) {
    if (dt == kF32) return reinterpret_cast<const float*>(p)[i];
    const u16 x = reinterpret_cast<const u16*>(p)[i];
    return dt == kBF16 ? Elem<kBF16>::to_f32(x) : Elem<kF16>::to_f32(x);
}

// Whether entry e is the first with its index.
__device__ inline bool first_of(const int* idx, int e) {
    for (int i = 0; i < e; ++i)
        if (idx[i] == idx[e]) return false;
    return true;
}

struct Sums4 {
    double a, p, z, z1;
};
__device__ inline Sums4 operator+(const Sums4& x, const Sums4& y) { return {x.a + y.a, x.p + y.p, x.z + y.z, x.z1 + y.z1}; }
template <int TB>
__device__ inline Sums4 block_sum(Sums4 v, Sums4* tmp) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v = v + Sums4{__shfl_xor(v.a, d), __shfl_xor(v.p, d), __shfl_xor(v.z, d), __shfl_xor(v.z1, d)};
    if constexpr (TB > 64) {
        if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = v;
        __syncthreads();
        v = tmp[0];
#pragma unroll
        for (int w = 1; w < TB / 64; ++w) v = v + tmp[w];
        __syncthreads();
    }
    return v;
}

// How the sum at temperature 1 (the cross entropy's) comes about: not at all or as the one at tau = 1, by exponentials of its own,
// or, where tau is 2 or 4, from squares of the others: e^z = (e^(z / 2))^2, one product or two for an exponential (each doubles
// the exponential's rounding). A second exponential makes the row's pass bound by instructions: 8192 x 50304 bf16 took 185 us
// with it and 145 without, 142 with the square.
enum Second { kNoSecond, kOwn, kSquare, kSquareTwice };
template <Second S2>
__device__ inline float second(float first) {
    const float q = first * first;
    return S2 == kSquareTwice ? q * q : q;
}

// 64 registers: eight blocks of 256 threads to a CU, so that 2048 rows are one round.
template <int DT, int TB, Second S2>
__global__ __launch_bounds__(TB, 8) void loss_fwd_kernel(Loss x) {
    using R = Row<DT>;
    using T = typename R::T;
    constexpr bool BOTH = S2 != kNoSecond;
    extern __shared__ uint32_t marks[];  // a bit per logit: the top set and the target
    __shared__ int idx[kMaxTop];
    __shared__ float zs[kMaxTop];
    __shared__ int bad, twice, target_in_top;
    __shared__ uint32_t zmost;  // the order of the top set's largest logit
    __shared__ Sums4 top_sums;  // (what the first wave needs at the end is not held in registers over the row)
    __shared__ double t_most;
    __shared__ float zt;
    __shared__ union {
        MaxSum sums[TB / 64];
        float f[TB / 64];
        double d[TB / 64];
        Sums4 d4[TB / 64];
    } tmp;
    const int r = blockIdx.x, tid = threadIdx.x, V = x.V, k = x.k;
    double* st = x.stats + (size_t)r * kStats;
    double& loss = x.stats[(size_t)gridDim.x * kStats + r];
    const long long target = x.targets ? x.targets[r] : 0;
    if (x.targets && target == kIgnore) {
        if (tid == 0) loss = 0.0;
        return;
    }
    const bool hard = x.hard(), target_ok = target >= 0 && target < V;
    const T* row = reinterpret_cast<const T*>(x.logits) + x.at.at(r);
    const int groups = (V + R::W - 1) / R::W;
    for (int i = tid; i < (groups * R::W + 31) / 32; i += TB) marks[i] = 0;
    if (tid == 0) bad = x.targets && !target_ok, twice = 0, target_in_top = 0, zmost = 0;
    __syncthreads();
    const double inv_tau = 1.0 / x.tau, ln2 = 0.6931471805599453;
    double tmax = x.rest ? (double)x.rest[r] : -INFINITY;
    for (int e = tid; e < k; e += TB) {
        const long long j = x.indices[(size_t)r * k + e];
        const bool ok = j >= 0 && j < V;
        idx[e] = ok ? (int)j : 0;
        zs[e] = R::one(row[idx[e]]);
        tmax = fmax(tmax, value_at(x.values, (long long)r * k + e, x.vdt) * inv_tau);
        if (!ok) {
            bad = 1;
            continue;
        }
        atomicMax(&zmost, Order<kF32>::of(__float_as_uint(zs[e])));
        const uint32_t bit = 1u << (j & 31), old = atomicOr(&marks[j >> 5], bit);
        if (hard && j == target) {  // (whose bit tells nothing: it is set below as well)
            if (atomicAdd(&target_in_top, 1) > 0) twice = 1;
        } else if (old & bit) {
            twice = 1;
        }
    }
    if (hard && tid == TB - 1 && target_ok) atomicOr(&marks[target >> 5], 1u << (target & 31));
    if (tid == 0) zt = hard && target_ok ? R::one(row[target]) : -INFINITY;
    __syncthreads();
    if (bad) {
        if (tid < kStats) st[tid] = tid == kTwice ? 0.0 : NAN;
        if (tid == 0) loss = NAN;
        return;
    }
    // The top set, in fp64: exponents relative to its (and the target's) largest logit, the teacher's to its largest term.
    const float near = Order<kF32>::K::value(zmost);
    {
        tmax = block_all<TB>(tmax, tmp.d, [](double a, double b) { return fmax(a, b); });
        const double base = base_of(fmaxf(near, zt));
        Sums4 top{0.0, 0.0, 0.0, 0.0};
        for (int e = tid; e < k; e += TB) {
            const double a = value_at(x.values, (long long)r * k + e, x.vdt) * inv_tau, z = zs[e], w = exp(a - tmax);
            top.a += w;
            if (!(w == 0.0)) top.p += w * (a - z * inv_tau);
            if (!twice || first_of(idx, e)) {
                top.z += exp((z - base) * inv_tau);
                if (hard) top.z1 += exp(z - base);
            }
        }
        top = block_sum<TB>(top, tmp.d4);
        if (tid == 0) top_sums = top, t_most = tmax;
        if constexpr (TB == 64) __syncthreads();  // (else the row's sums have one)
    }

    // The row without what is marked. Exponents are in powers of two relative to 2^b, the whole number b next to the exponent of
    // the top set's largest logit (so that z c - b is rounded once).
    const float b = rintf(near * x.c), b1 = S2 == kSquare ? 2 * b : S2 == kSquareTwice ? 4 * b : rintf(near * kL2e);
    float s = 0.f, s1 = 0.f;
    const uint8_t* bytes = reinterpret_cast<const uint8_t*>(marks);
    auto marks_of = [&](int i) { return R::W == 8 ? bytes[i] : (bytes[i >> 1] >> (4 * (i & 1))) & 15; };
    auto take_group = [&](u32x4 raw, int m) {
        float v[R::W];
        R::widen(raw, v);
        if (m) {
#pragma unroll
            for (int e = 0; e < R::W; ++e) v[e] = (m >> e) & 1 ? -INFINITY : v[e];
        }
#pragma unroll
        for (int e = 0; e < R::W; ++e) {
            const float y = __builtin_amdgcn_exp2f(fmaf(v[e], x.c, -b));
            s += y;
            if constexpr (S2 == kOwn) s1 += __builtin_amdgcn_exp2f(fmaf(v[e], kL2e, -b1));
            if constexpr (S2 == kSquare || S2 == kSquareTwice) s1 += second<S2>(y);
        }
    };
    {
        constexpr int U = 4;  // loads under way
        const int whole = V / R::W;
        int i = tid;
        for (; i + (U - 1) * TB < whole; i += U * TB) {
            u32x4 raw[U];
#pragma unroll
            for (int u = 0; u < U; ++u) raw[u] = group_at<DT>(row, i + u * TB, V);
#pragma unroll
            for (int u = 0; u < U; ++u) take_group(raw[u], marks_of(i + u * TB));
        }
        for (; i < groups; i += TB) take_group(group<DT>(row, i, V), marks_of(i));
    }
    s = block_all<TB>(s, tmp.f, [](float a, float b) { return a + b; });
    if constexpr (BOTH) s1 = block_all<TB>(s1, tmp.f, [](float a, float b) { return a + b; });
    // The sums times e^from (c is log2(e) / tau rounded: what that puts on the exponents near b comes off again).
    const double off = near * (inv_tau - (double)x.c * ln2);
    double from = ln2 * b + off, from1 = S2 == kOwn ? ln2 * b1 + near * (1.0 - (double)kL2e * ln2) : ln2 * b1 + off * x.tau;
    if (!(stands(s) && (!BOTH || stands(s1)))) {
        // Far from the top set's: relative to their own largest.
        MaxSum a{-INFINITY, 0.f, 0.f};
        for (int i = tid; i < groups; i += TB) {
            float v[R::W];
            R::widen(group<DT>(row, i, V), v);
            const int m = marks_of(i);
#pragma unroll
            for (int e = 0; e < R::W; ++e) v[e] = (m >> e) & 1 ? -INFINITY : v[e];
            take<BOTH, R::W>(a, v, x.c);
        }
        a = block_merge<TB, BOTH>(a, tmp.sums, x.c);
        s = a.m == INFINITY ? NAN : a.s, s1 = a.s1;  // (as softmax has it: inf - inf)
        from = base_of(a.m) * inv_tau, from1 = base_of(a.m);
    }
    if constexpr (!BOTH) s1 = s, from1 = from;  // (read only where the temperature is 1)
    if (tid >= 64) return;
    const Sums4 top = top_sums;
    const float z_target = zt, zmax = fmaxf(near, z_target);
    const double base = base_of(zmax), z_soft = z_target * inv_tau;
    // (-inf where all of these are: the others' sum alone says then what the joined ones are relative to)
    const double at1 = zmax == -INFINITY ? -INFINITY : base, at = at1 * inv_tau;
    tmax = t_most;

    // All that is joined: logarithms and exponentials one a lane, since each takes as long as 64 of them.
    auto lane_of = [](double v, int lane) { return __shfl(v, lane); };
    const double rest = x.rest ? (double)x.rest[r] : -INFINITY, ls = log((double)(tid == 0 ? s : s1));
    const double Ls = s == 0.f ? -INFINITY : from + lane_of(ls, 0), Ls1 = s == 0.f ? -INFINITY : from1 + lane_of(ls, 1);
    const bool alone = hard && !target_in_top;  // (then the target is one of the others, but not in their sum)
    const double to = fmax(at, Ls), to1 = fmax(at1, Ls1), to_r = alone ? fmax(Ls, z_soft) : Ls;
    const double arg = tid == 0   ? Ls - to
                       : tid == 1 ? Ls1 - to1
                       : tid == 2 ? z_soft - to
                       : tid == 3 ? z_target - to1
                       : tid == 4 ? rest - tmax
                       : tid == 5 ? at - to
                       : tid == 6 ? at1 - to1
                       : tid == 7 ? Ls - to_r
                                  : z_soft - to_r;
    const double ex = exp(arg);
    const double w = x.rest ? lane_of(ex, 4) : 0.0, A = top.a + w;
    const double Z = top.z * lane_of(ex, 5) + lane_of(ex, 0) + (alone ? lane_of(ex, 2) : 0.0);
    const double Z1 = top.z1 * lane_of(ex, 6) + lane_of(ex, 1) + (alone ? lane_of(ex, 3) : 0.0);
    const double lg = log(tid == 0 ? Z : tid == 1 ? Z1 : tid == 2 ? A : lane_of(ex, 7) + lane_of(ex, 8));
    const double L = to + lane_of(lg, 0), L1 = hard ? to1 + lane_of(lg, 1) : 0.0, Lt = tmax + lane_of(lg, 2);
    const double Lr = to_r == -INFINITY ? to_r : alone ? to_r + lane_of(lg, 3) : Ls;
    if (tid != 0) return;
    double P = top.p;
    if (!(w == 0.0)) P += w * (rest - Lr);
    // The gradient's exponentials, at both temperatures, are relative to one logit, which has to lie near the others' largest: for
    // temperatures above 1 their logsumexp at 1, below 1 the one at tau times tau (the lower one: the other lies up to tau ln V,
    // or ln V, above, past fp32's exponents for a tau of 9). (No others: the target's, or the top set's, so that the factors of
    // exponentials that are 0 stay finite.)
    const float own = (float)(BOTH ? fmin(Ls * x.tau, Ls1) : Ls * x.tau), no_own = alone && fabsf(z_target) < INFINITY ? z_target : (float)base;
    st[kL] = L, st[kL1] = L1, st[kLt] = Lt, st[kLr] = Lr, st[kPr] = w / A, st[kBase] = fabsf(own) < INFINITY ? own : no_own, st[kTwice] = twice;
    double v = 0.0;
    if (zmax == INFINITY) v = st[kL] = NAN;  // (inf - inf again)
    if (x.weight > 0.0) v += x.weight * x.tau * x.tau * (P / A - Lt + L);
    if (hard) v += (1.0 - x.weight) * (L1 - z_target);
    loss = v;
}

// loss = the rows' sum / n and 1 / n, n the rows that count: one block, in a fixed order.
__global__ __launch_bounds__(1024) void loss_mean_kernel(const long long* __restrict__ targets, double* __restrict__ stats, float* __restrict__ loss, int R) {
    const double* rows = stats + (size_t)R * kStats;
    double s = 0.0;
    int n = 0;
    for (int i = threadIdx.x; i < R; i += 8 * 1024) {  // (8 rows under way)
        double v[8];
        bool on[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int r = i + u * 1024;
            on[u] = r < R && (!targets || targets[r] != kIgnore);
            v[u] = r < R ? rows[r] : 0.0;
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) s += v[u], n += on[u];
    }
    __shared__ double tmp[16];
    __shared__ int tmpn[16];
    s = block_all<1024>(s, tmp, [](double a, double b) { return a + b; });
    n = block_all<1024>(n, tmpn, [](int a, int b) { return a + b; });
    if (threadIdx.x == 0) {
        *loss = (float)(s / n);
        stats[(size_t)R * (kStats + 1)] = 1.0 / n;
    }
}

template <int DT, int TB, Second S2>
__global__ __launch_bounds__(TB, 8) void loss_bwd_kernel(Loss x, const float* __restrict__ grad, void* __restrict__ dlogits) {
    using R = Row<DT>;
    using T = typename R::T;
    __shared__ int idx[kMaxTop];
    __shared__ int target_in_top;
    // (from the last row on, which the forward has read last: what the caches still hold of it is not read from memory again)
    const int r = gridDim.x - 1 - blockIdx.x, tid = threadIdx.x, V = x.V, k = x.k;
    T* dst = reinterpret_cast<T*>(dlogits) + (size_t)r * V;
    const int whole = V / R::W, tail = whole * R::W;
    const long long target = x.targets ? x.targets[r] : 0;
    if (x.targets && target == kIgnore) {
        for (int i = tid; i < whole; i += TB) store_any<DT>(dst + i * R::W, u32x4{});
        if (tail + tid < V) dst[tail + tid] = (T)0;
        return;
    }
    const bool hard = x.hard(), soft = x.weight > 0.0;
    const T* row = reinterpret_cast<const T*>(x.logits) + x.at.at(r);
    const double* st = x.stats + (size_t)r * kStats;
    const double inv_tau = 1.0 / x.tau, L = st[kL], L1 = st[kL1], Lr = st[kLr], base = st[kBase];
    // (where the student's rest is empty, its loss infinite, no logit has a share of the teacher's)
    const double p_rest = Lr == -INFINITY && st[kPr] > 0.0 ? 0.0 : st[kPr];
    const double g = (double)grad[0] * x.stats[(size_t)gridDim.x * (kStats + 1)], gs = soft ? x.weight * x.tau * g : 0.0, gh = hard ? (1.0 - x.weight) * g : 0.0;
    // q_j f_j of a logit outside the top set, which is q_j - p_rest times its share of the rest.
    auto outside = [&](double z) {
        const double share = p_rest == 0.0 ? 0.0 : p_rest * exp(z * inv_tau - Lr);
        return gs * (exp(z * inv_tau - L) - share);
    };
    // Every logit as one of those, relative to one of their size: the rest may lie far below the top set.
    float A = soft ? (float)outside(base) : 0.f;
    const float B = hard ? (float)(gh * exp(base - L1)) : 0.f, b = (float)base;
    if constexpr (S2 == kNoSecond) A += B;  // (there is B only where the temperature is 1)
    if (L != L) A = NAN;          // an index or target out of range, or a NaN or +inf in the row
    auto of = [&](float z) {
        const float d = z - b, y = __builtin_amdgcn_exp2f(d * x.c);
        if constexpr (S2 == kNoSecond)
            return A * y;
        else
            return A * y + B * (S2 == kOwn ? __builtin_amdgcn_exp2f(d * kL2e) : second<S2>(y));
    };
    for (int i = tid; i < whole; i += TB) {
        float v[R::W];
        R::widen(load_any<DT>(row + i * R::W), v);
#pragma unroll
        for (int e = 0; e < R::W; ++e) v[e] = of(v[e]);
        store_any<DT>(dst + i * R::W, R::narrow(v));
    }
    if (tail + tid < V) dst[tail + tid] = R::round(of(R::one(row[tail + tid])));
    if (L != L) return;
    // Then the top set and the target, over what was stored.
    for (int e = tid; e < k; e += TB) {
        const long long j = x.indices[(size_t)r * k + e];
        idx[e] = j >= 0 && j < V ? (int)j : -1;  // (statistics of other indices lead to no access outside the row)
    }
    if (tid == 0) target_in_top = 0;
    __syncthreads();
    const bool twice = st[kTwice] != 0.0;
    for (int e = tid; e < k; e += TB) {
        const int j = idx[e];
        if (j < 0) continue;
        if (hard && j == target) target_in_top = 1;
        if (twice && !first_of(idx, e)) continue;
        const double z = R::one(row[j]);
        double v = 0.0;
        if (soft) {
            double p = 0.0;
            for (int i = e; i < (twice ? k : e + 1); ++i)
                if (idx[i] == j) p += exp(value_at(x.values, (long long)r * k + i, x.vdt) * inv_tau - st[kLt]);
            v = gs * (exp(z * inv_tau - L) - p);
        }
        if (hard) v += gh * (exp(z - L1) - (j == target ? 1.0 : 0.0));
        dst[j] = R::round((float)v);
    }
    __syncthreads();
    if (hard && tid == 0 && !target_in_top && target >= 0 && target < V) {
        const double z = R::one(row[target]);
        dst[target] = R::round((float)((soft ? outside(z) : 0.0) + gh * (exp(z - L1) - 1.0)));
    }
}

// ------------------------------------------------------------------------------------------
// Host side.
// ------------------------------------------------------------------------------------------
thread_local std::string g_err;

int fail(const char* what) {
    g_err = what;
    return -1;
}

int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        g_err = std::string(what) + " launch failed: " + hipGetErrorString(e);
        return (int)e;
    }
    return 0;
}

int check(int64_t T, int64_t sb, int64_t st, int64_t R, int64_t V, int64_t k, double temperature, int dtype, const void* logits) {
    g_err.clear();
    if (R < 1 || R >= (1 << 22) || V < 1 || V > kMaxVocab || T < 1 || T > R) return fail("invalid sizes");
    if (k < 1 || k > V || k > kMaxTop) return fail("k must be in [1, min(V, 512)]");
    if (sb < 0 || st < 0 || sb >= ((int64_t)1 << 40) || st >= ((int64_t)1 << 40)) return fail("invalid strides");
    if (!(temperature >= 1e-4 && temperature <= 1e4)) return fail("temperature must be in [1e-4, 1e4]");
    if (dtype != kF16 && dtype != kBF16 && dtype != kF32) return fail("dtype must be float16, bfloat16 or float32");
    if ((uintptr_t)logits % (dtype == kF32 ? 4 : 2)) return fail("logits must be aligned to their type");
    return 0;
}

template <typename F>
int by_dtype(int dtype, F f) {
    return dtype == kBF16 ? f(std::integral_constant<int, kBF16>()) : dtype == kF16 ? f(std::integral_constant<int, kF16>())
                                                                                    : f(std::integral_constant<int, kF32>());
}

size_t mark_bytes(int64_t V) { return (size_t)((V + 7 + 31) / 32) * 4; }

}  // namespace

NNDIS_API const char* nn_distill_last_error(void) { return g_err.c_str(); }

NNDIS_API int nn_top_logits(const void* logits, int64_t T, int64_t sb, int64_t st, void* values, int64_t* indices, float* rest, int64_t R,
                            int64_t V, int64_t k, double temperature, int dtype, void* stream) {
    if (int e = check(T, sb, st, R, V, k, temperature, dtype, logits)) return e;
    if (!logits || !values || !indices || !rest) return fail("null pointer argument");
    return by_dtype(dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        auto go = [&](auto kern, int threads) {
            kern<<<dim3((unsigned)R), dim3(threads), 0, (hipStream_t)stream>>>(logits, Layout{sb, st, (int)T}, values, (long long*)indices, rest, (int)V,
                                                                               (int)k, (float)(1.4426950408889634 / temperature), 1.0 / temperature);
            return launched("top_kernel");
        };
        const int64_t groups = (V + Row<DT>::W - 1) / Row<DT>::W;  // of 16 bytes, held by the block's threads
        // One wave a row up to 256 groups (groups past the row's end take as long as others: 468000 x 512 bf16, k = 6, 733 us with
        // 4 a thread).
        return groups <= 64          ? go(top_kernel<DT, 64, 1>, 64)
               : groups <= 2 * 64    ? go(top_kernel<DT, 64, 2>, 64)
               : groups <= 4 * 64    ? go(top_kernel<DT, 64, 4>, 64)
               : groups <= 4 * 256   ? go(top_kernel<DT, 256, 4>, 256)
               : groups <= 8 * 512   ? go(top_kernel<DT, 512, 8>, 512)
               : groups <= 13 * 512  ? go(top_kernel<DT, 512, 13>, 512)
               : groups <= 16 * 512  ? go(top_kernel<DT, 512, 16>, 512)
               : groups <= 16 * 1024 ? go(top_kernel<DT, 1024, 16>, 1024)
                                     : go(top_kernel<DT, 1024, 0>, 1024);
    });
}

NNDIS_API size_t nn_distill_stats_size(int64_t R) { return R < 1 ? 0 : (size_t)R * (kStats + 1) + 1; }

namespace {
int check_loss(int64_t T, int64_t sb, int64_t st, int64_t R, int64_t V, int64_t k, double temperature, double weight, int dtype, int value_dtype,
               const void* logits) {
    if (int e = check(T, sb, st, R, V, k, temperature, dtype, logits)) return e;
    if (!(weight >= 0.0 && weight <= 1.0)) return fail("weight must be in [0, 1]");
    if (value_dtype != kF16 && value_dtype != kBF16 && value_dtype != kF32) return fail("dtype must be float16, bfloat16 or float32");
    return 0;
}
// Launches a loss kernel: 64 threads for a short row, 256 for a long one.
template <template <int, int, Second> class Kernel, typename F>
int by_row(const Loss& x, int dtype, F go) {
    const Second two = !x.targets || x.weight >= 1.0 || x.tau == 1.0 ? kNoSecond : x.tau == 2.0 ? kSquare : x.tau == 4.0 ? kSquareTwice : kOwn;
    return by_dtype(dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        auto of = [&](auto s2) {
            constexpr Second S2 = decltype(s2)::value;
            return x.V <= 2048 ? go(Kernel<DT, 64, S2>::fn, 64) : go(Kernel<DT, 256, S2>::fn, 256);
        };
        switch (two) {
            case kOwn: return of(std::integral_constant<Second, kOwn>());
            case kSquare: return of(std::integral_constant<Second, kSquare>());
            case kSquareTwice: return of(std::integral_constant<Second, kSquareTwice>());
            default: return of(std::integral_constant<Second, kNoSecond>());
        }
    });
}
template <int DT, int TB, Second S2>
struct Fwd {
    static constexpr auto fn = loss_fwd_kernel<DT, TB, S2>;
};
template <int DT, int TB, Second S2>
struct Bwd {
    static constexpr auto fn = loss_bwd_kernel<DT, TB, S2>;
};
}  // namespace

NNDIS_API int nn_distill_fwd(const void* logits, int64_t T, int64_t sb, int64_t st, const void* values, const int64_t* indices, const float* rest,
                             const int64_t* targets, float* loss, double* stats, int64_t R, int64_t V, int64_t k, double temperature,
                             double weight, int dtype, int value_dtype, void* stream) {
    if (int e = check_loss(T, sb, st, R, V, k, temperature, weight, dtype, value_dtype, logits)) return e;
    if (!logits || !values || !indices || !loss || !stats) return fail("null pointer argument");
    const Loss x{logits, Layout{sb, st, (int)T}, values, (const long long*)indices, rest, (const long long*)targets, stats, (int)V, (int)k, value_dtype,
                 (float)(1.4426950408889634 / temperature), temperature, weight};
    if (int e = by_row<Fwd>(x, dtype, [&](auto kern, int threads) {
            kern<<<dim3((unsigned)R), dim3(threads), mark_bytes(V), (hipStream_t)stream>>>(x);
            return launched("loss_fwd_kernel");
        }))
        return e;
    loss_mean_kernel<<<dim3(1), dim3(1024), 0, (hipStream_t)stream>>>((const long long*)targets, stats, loss, (int)R);
    return launched("loss_mean_kernel");
}

NNDIS_API int nn_distill_bwd(const float* grad, const void* logits, int64_t T, int64_t sb, int64_t st, const void* values,
                             const int64_t* indices, const int64_t* targets, const double* stats, void* dlogits, int64_t R, int64_t V, int64_t k,
                             double temperature, double weight, int dtype, int value_dtype, void* stream) {
    if (int e = check_loss(T, sb, st, R, V, k, temperature, weight, dtype, value_dtype, logits)) return e;
    if ((uintptr_t)dlogits % (dtype == kF32 ? 4 : 2)) return fail("dlogits must be aligned to their type");
    if (!grad || !logits || !values || !indices || !stats || !dlogits) return fail("null pointer argument");
    const Loss x{logits, Layout{sb, st, (int)T}, values, (const long long*)indices, nullptr, (const long long*)targets, const_cast<double*>(stats), (int)V,
                 (int)k, value_dtype, (float)(1.4426950408889634 / temperature), temperature, weight};
    return by_row<Bwd>(x, dtype, [&](auto kern, int threads) {
        kern<<<dim3((unsigned)R), dim3(threads), 0, (hipStream_t)stream>>>(x, grad, dlogits);
        return launched("loss_bwd_kernel");
    });
}
