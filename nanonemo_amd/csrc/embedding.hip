// Embedding lookup with a scale, and its gradient by sorted tokens, for MI355X (gfx950).
//
//   forward    out[m] = s * W[idx[m]]
//   backward   dW[v] = s * sum over the m with idx[m] = v of dy[m]
//
// Backward. The positions are sorted by token (a stable radix sort, so that equal tokens keep their order), the sorted
// list is cut into chunks of equal length, and a wave sums a chunk's rows of dy token by token. A token whose rows lie in
// one chunk is stored at once; the sums of one that is cut by chunk borders go to the workspace as fp32 and are joined by
// fixup_kernel: in chunk order, or for a long run by 16 waves, each every 16th, and the waves' in order. The work is even
// whatever the tokens are (a batch of one repeated token is as many waves as any other), there are no atomics on values, and the
// order of every sum is fixed by the tokens and the sizes: the result is bit-reproducible.
// Rows of dW without a token are zeroed by further blocks of the sort's launches, which leave the memory idle otherwise.
// Bound by HBM: dy is read once and dW written once.
//
// Built with NaN semantics: a token out of range gives a NaN row.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <string>

#include "nanonemo_embedding.h"
#include "rows.h"

#define NNEMB_API extern "C" __attribute__((visibility("default")))

namespace {

constexpr int kThreads = 256;

// ------------------------------------------------------------------------------------------
// Forward: a thread owns kFwdUnits 16-byte units of the output (or single values where rows are not whole units).
// ------------------------------------------------------------------------------------------
constexpr int kFwdUnits = 4;

// UNIT: values of a unit, Row<DT>::W or 1. PAST: stored past the caches.
template <int DT, int UNIT, bool PAST, typename I>
__global__ __launch_bounds__(kThreads) void fwd_kernel(const void* __restrict__ weight, const I* __restrict__ idx,
                                                       void* __restrict__ out, long long units, int per_row, int V, float scale) {
    using R = Row<DT>;
    using T = typename R::T;
    const T* w = reinterpret_cast<const T*>(weight);
    T* o = reinterpret_cast<T*>(out);
    const long long first = (long long)blockIdx.x * (kThreads * kFwdUnits);
    const long long row0 = first / per_row;  // (uniform; the divisions below are 32-bit)
    const unsigned off0 = (unsigned)(first - row0 * per_row);
    long long src[kFwdUnits], dst[kFwdUnits];
    bool on[kFwdUnits], bad[kFwdUnits];
#pragma unroll
    for (int k = 0; k < kFwdUnits; ++k) {
        const unsigned i = off0 + k * kThreads + threadIdx.x;
        const unsigned r = i / (unsigned)per_row, c = i - r * per_row;
        dst[k] = first + k * kThreads + threadIdx.x;
        on[k] = dst[k] < units;
        const long long t = on[k] ? (long long)idx[row0 + r] : 0;
        bad[k] = t < 0 || t >= V;
        src[k] = bad[k] ? 0 : t * per_row + c;
    }
    if constexpr (UNIT == 1) {
        T v[kFwdUnits];
#pragma unroll
        for (int k = 0; k < kFwdUnits; ++k) v[k] = w[on[k] ? src[k] : 0];
#pragma unroll
        for (int k = 0; k < kFwdUnits; ++k)
            if (on[k]) o[dst[k]] = R::round(bad[k] ? NAN : R::one(v[k]) * scale);
    } else {
        u32x4 raw[kFwdUnits];
#pragma unroll
        for (int k = 0; k < kFwdUnits; ++k) raw[k] = R::raw(w + (on[k] ? src[k] : 0) * UNIT);
#pragma unroll
        for (int k = 0; k < kFwdUnits; ++k) {
            if (!on[k]) continue;
            float v[R::W];
            R::widen(raw[k], v);
#pragma unroll
            for (int e = 0; e < R::W; ++e) v[e] = bad[k] ? NAN : v[e] * scale;
            if constexpr (PAST)
                __builtin_nontemporal_store(R::narrow(v), reinterpret_cast<u32x4*>(o + dst[k] * UNIT));
            else
                R::store(o + dst[k] * UNIT, v);
        }
    }
}

// ------------------------------------------------------------------------------------------
// The sort: (token, position) pairs by token, least significant digits first. Tokens that take no part have the key V and
// end up last.
// ------------------------------------------------------------------------------------------
constexpr int kDigit = 9, kBins = 1 << kDigit;  // 18-bit vocabularies in two passes
constexpr int kSortThreads = kBins, kSortWaves = kSortThreads / 64;
constexpr int kItems = 2, kSub = kSortThreads * kItems;  // entries of a block's step
constexpr int kMostSortBlocks = 128;                     // (every block reads every block's counts)

// The lanes of the wave with this lane's digit, among those that are on.
__device__ inline uint64_t same_digit(int d, bool on) {
    uint64_t m = __ballot(on);
#pragma unroll
    for (int b = 0; b < kDigit; ++b) {
        const bool bit = (d >> b) & 1;
        const uint64_t v = __ballot(bit);
        m &= bit ? v : ~v;
    }
    return m;
}

struct Pairs {
    const void* idx;      // the first pass reads the tokens
    const uint32_t* key;  // later ones what the pass before wrote
    const int* pos;
    long long pad;
    int V, shift;
};
template <typename I, bool FIRST>
__device__ inline uint32_t key_at(const Pairs& p, int i) {
    if constexpr (FIRST) {
        const long long t = reinterpret_cast<const I*>(p.idx)[i];
        return t >= 0 && t < p.V && t != p.pad ? (uint32_t)t : (uint32_t)p.V;
    } else {
        return p.key[i];
    }
}

// Zeros of dW by the blocks of a launch that do not sort: units [begin, end) of 16 bytes, and after the last unit the
// matrix's last few values.
struct Fill {
    u32x4* at;
    long long begin, end;
    u16* tail;
    int ntail;
};
__device__ inline void fill(const Fill& f, int block, int blocks) {
    for (long long i = f.begin + (long long)block * blockDim.x + threadIdx.x; i < f.end; i += (long long)blocks * blockDim.x) __builtin_nontemporal_store(u32x4{}, f.at + i);
    if (block == 0 && (int)threadIdx.x < f.ntail) f.tail[threadIdx.x] = 0;
}
__global__ __launch_bounds__(kSortThreads) void fill_kernel(Fill f) { fill(f, blockIdx.x, gridDim.x); }

// Counts of this pass's digits in each block's entries [block * per, + per).
template <typename I, bool FIRST>
__global__ __launch_bounds__(kSortThreads) void count_kernel(Pairs p, int M, int per, int nb, int* __restrict__ counts, Fill f) {
    if ((int)blockIdx.x >= nb) return fill(f, blockIdx.x - nb, gridDim.x - nb);
    __shared__ int h[kBins];
    const int tid = threadIdx.x, lane = tid & 63;
    h[tid] = 0;
    __syncthreads();
    const long long begin = (long long)blockIdx.x * per;
    const int end = (int)min((long long)M, begin + per);
    for (long long s = begin; s < end; s += kSortThreads) {
        const long long i = s + tid;
        const bool on = i < end;
        const int d = on ? (key_at<I, FIRST>(p, (int)i) >> p.shift) & (kBins - 1) : 0;
        const uint64_t m = same_digit(d, on);
        if (on && lane == __ffsll((unsigned long long)m) - 1) atomicAdd(&h[d], __popcll(m));
    }
    __syncthreads();
    counts[blockIdx.x * kBins + tid] = h[tid];
}

// Every entry to its place: digits in order, within a digit the blocks in order, within a block the entries in order.
template <typename I, bool FIRST>
__global__ __launch_bounds__(kSortThreads) void place_kernel(Pairs p, int M, int per, int nb, const int* __restrict__ counts,
                                                             uint32_t* __restrict__ key_out, int* __restrict__ pos_out, Fill f) {
    if ((int)blockIdx.x >= nb) return fill(f, blockIdx.x - nb, gridDim.x - nb);
    __shared__ int wave_count[kSortWaves][kBins];
    __shared__ int wave_all[kSortWaves][kBins];
    __shared__ int wave_total[kSortWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // Digit tid's first place for this block: all smaller digits' entries, and the blocks' before this one. Every wave adds up an
    // eighth of the blocks' counts, eight digits a lane, with all loads under way (one after the other they took 10 us of 128
    // blocks).
    {
        constexpr int PER = kBins / 64, EACH = kMostSortBlocks / kSortWaves;
        int before[PER] = {}, total[PER] = {};
#pragma unroll
        for (int b = 0; b < EACH; ++b) {
            const int block = b * kSortWaves + wave, on = block < nb, earlier = block < (int)blockIdx.x;
            const int4* c = reinterpret_cast<const int4*>(counts + min(block, nb - 1) * kBins + lane * PER);
#pragma unroll
            for (int q = 0; q < PER / 4; ++q) {
                const int4 v = c[q];
                const int e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    total[4 * q + i] += on ? e[i] : 0;
                    before[4 * q + i] += earlier ? e[i] : 0;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) wave_count[wave][lane * PER + i] = before[i], wave_all[wave][lane * PER + i] = total[i];
    }
    __syncthreads();
    int before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) before += wave_count[w][tid], total += wave_all[w][tid];
    int scan = total;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int t = __shfl_up(scan, d);
        scan += lane >= d ? t : 0;
    }
    if (lane == 63) wave_total[wave] = scan;
    __syncthreads();
    int base = scan - total + before;
    for (int w = 0; w < wave; ++w) base += wave_total[w];

    const long long begin = (long long)blockIdx.x * per;
    const int end = (int)min((long long)M, begin + per);
    for (long long s = begin; s < end; s += kSub) {
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) wave_count[w][tid] = 0;
        __syncthreads();
        uint32_t key[kItems];
        int pos[kItems], rank[kItems];
        bool on[kItems];
#pragma unroll
        for (int k = 0; k < kItems; ++k) {  // a wave's items are consecutive runs of 64 entries
            const long long i = s + wave * (64 * kItems) + k * 64 + lane;
            on[k] = i < end;
            key[k] = on[k] ? key_at<I, FIRST>(p, (int)i) : 0;
            pos[k] = FIRST ? (int)i : on[k] ? p.pos[i] : 0;
        }
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
            const int d = (key[k] >> p.shift) & (kBins - 1);
            const uint64_t m = same_digit(d, on[k]);
            const int leader = m ? __ffsll((unsigned long long)m) - 1 : 0;
            int old = 0;
            if (on[k] && lane == leader) old = atomicAdd(&wave_count[wave][d], __popcll(m));
            rank[k] = __shfl(old, leader) + __popcll(m & ((1ull << lane) - 1));
        }
        __syncthreads();
        int run = base;
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) {
            const int c = wave_count[w][tid];
            wave_count[w][tid] = run;
            run += c;
        }
        base = run;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
            if (!on[k]) continue;
            const int at = wave_count[wave][(key[k] >> p.shift) & (kBins - 1)] + rank[k];
            key_out[at] = key[k];
            pos_out[at] = pos[k];
        }
        __syncthreads();
    }
}

// Up to kSmall entries: one block sorts them in LDS, all passes in one launch, while the others zero dW. The whole gradient of
// 8192 x 768 fp32 into 50304 rows: 46 us, with the four launches above 49 (and three more launches for the host); of 16384 tokens
// 72 and 61: there the one block takes longer than the zeros.
constexpr int kSmallThreads = 1024, kSmallWaves = kSmallThreads / 64, kSmallItems = 8, kSmall = kSmallThreads * kSmallItems;
template <typename I>
__global__ __launch_bounds__(kSmallThreads) void sort_small_kernel(Pairs p, int M, int passes, uint32_t* __restrict__ key_out, int* __restrict__ pos_out,
                                                                   Fill f) {
    if (blockIdx.x > 0) return fill(f, blockIdx.x - 1, gridDim.x - 1);
    __shared__ uint32_t keys[kSmall];
    __shared__ u16 positions[kSmall];
    __shared__ int wave_count[kSmallWaves][kBins];
    __shared__ int wave_total[kBins / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int items = (M + kSmallThreads - 1) / kSmallThreads, first = wave * 64 * items + lane;  // entries first + 64 i
    uint32_t key[kSmallItems];
    int pos[kSmallItems], rank[kSmallItems];
#pragma unroll
    for (int i = 0; i < kSmallItems; ++i) {
        const int e = first + 64 * i;
        const bool on = i < items && e < M;
        key[i] = on ? key_at<I, true>(p, e) : 0;
        pos[i] = e;
    }
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = pass * kDigit;
        for (int i = tid; i < kSmallWaves * kBins; i += kSmallThreads) (&wave_count[0][0])[i] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kSmallItems; ++i) {
            if (i >= items) continue;
            const bool on = first + 64 * i < M;
            const int d = (key[i] >> shift) & (kBins - 1);
            const uint64_t m = same_digit(d, on);
            const int leader = m ? __ffsll((unsigned long long)m) - 1 : 0;
            int old = 0;
            if (on && lane == leader) old = atomicAdd(&wave_count[wave][d], __popcll(m));
            rank[i] = __shfl(old, leader) + __popcll(m & ((1ull << lane) - 1));
        }
        __syncthreads();
        int total = 0, scan = 0;
        if (tid < kBins) {  // (whole waves)
#pragma unroll
            for (int w = 0; w < kSmallWaves; ++w) total += wave_count[w][tid];
            scan = total;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int t = __shfl_up(scan, d);
                scan += lane >= d ? t : 0;
            }
            if (lane == 63) wave_total[wave] = scan;
        }
        __syncthreads();
        if (tid < kBins) {
            int run = scan - total;
            for (int w = 0; w < wave; ++w) run += wave_total[w];
#pragma unroll
            for (int w = 0; w < kSmallWaves; ++w) {
                const int c = wave_count[w][tid];
                wave_count[w][tid] = run;
                run += c;
            }
        }
        __syncthreads();
        const bool last = pass + 1 == passes;
#pragma unroll
        for (int i = 0; i < kSmallItems; ++i) {
            if (i >= items || first + 64 * i >= M) continue;
            const int at = wave_count[wave][(key[i] >> shift) & (kBins - 1)] + rank[i];
            if (last) {
                key_out[at] = key[i];
                pos_out[at] = pos[i];
            } else {
                keys[at] = key[i];
                positions[at] = (u16)pos[i];
            }
        }
        if (last) break;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kSmallItems; ++i) {
            const int e = first + 64 * i;
            if (i < items && e < M) key[i] = keys[e], pos[i] = positions[e];
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------------------
// The sums. VEC values of a lane, 64 VEC columns of a wave: 4, or 1 where rows are not whole groups of 4. dy is not needed again,
// and its loads do not stay in the caches.
// ------------------------------------------------------------------------------------------
template <int DT, int VEC>
__device__ inline void load_vec(const typename Row<DT>::T* p, float* v) {
    if constexpr (VEC == 1) {
        v[0] = Row<DT>::one(*p);
    } else if constexpr (DT == kF32) {
        const f32x4 x = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p));
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = x[e];
    } else {
        const u16x4 x = __builtin_nontemporal_load(reinterpret_cast<const u16x4*>(p));
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = Elem<DT>::to_f32(x[e]);
    }
}
template <int DT, int VEC>
__device__ inline void store_vec(typename Row<DT>::T* p, const float* v, float scale) {
    if constexpr (VEC == 1) {
        *p = Row<DT>::round(v[0] * scale);
    } else if constexpr (DT == kF32) {
        *reinterpret_cast<f32x4*>(p) = f32x4{v[0] * scale, v[1] * scale, v[2] * scale, v[3] * scale};
    } else {
        *reinterpret_cast<u32x2*>(p) = u32x2{Elem<DT>::pack2(v[0] * scale, v[1] * scale), Elem<DT>::pack2(v[2] * scale, v[3] * scale)};
    }
}

struct Sums {
    const uint32_t* key;  // sorted tokens, and their positions
    const int* pos;
    float* part;          // [chunks][2][ld]: a chunk's sum of the token that began before it, and of the one that goes on after it
    int M, V, N, ld, chunk, slabs;
    float scale;
};

// A wave per chunk and 64 VEC columns. 131072 x 768 bf16 (201 MB of dy): 41 us, with cached loads 62.
template <int DT, int VEC>
__global__ __launch_bounds__(kThreads) void sum_kernel(Sums a, const void* __restrict__ dy_, void* __restrict__ dw_, long long waves) {
    using T = typename Row<DT>::T;
    constexpr int U = 16;  // rows in flight
    const T* dy = reinterpret_cast<const T*>(dy_);
    T* dw = reinterpret_cast<T*>(dw_);
    const long long id = (long long)blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (id >= waves) return;
    const int c = (int)(id / a.slabs), lane = threadIdx.x & 63, col = ((int)(id - (long long)c * a.slabs) * 64 + lane) * VEC;
    const int lo = c * a.chunk, most = min(a.chunk, a.M - lo);
    const uint32_t key = lane < most ? a.key[lo + lane] : a.V;
    const int pos = lane < most ? a.pos[lo + lane] : 0;
    const int n = __popcll(__ballot(key < (uint32_t)a.V));
    if (n == 0) return;
    const uint32_t prev = lo > 0 ? a.key[lo - 1] : (uint32_t)a.V, next = lo + most < a.M ? a.key[lo + most] : (uint32_t)a.V;
    const bool mine = col < a.N;
    const int at = mine ? col : 0;  // (lanes past the last column read the first and store nothing)
    float acc[VEC];
    uint32_t cur = __builtin_amdgcn_readlane(key, 0);
    bool head = cur == prev;  // whether the token began before this chunk
    float* part = a.part + (size_t)c * 2 * a.ld + at;
    auto partial = [&](int which) {
        if (!mine) return;
#pragma unroll
        for (int e = 0; e < VEC; ++e) part[(size_t)which * a.ld + e] = acc[e];
    };
    auto store = [&]() {
        if (mine) store_vec<DT, VEC>(dw + (size_t)cur * a.N + at, acc, a.scale);
    };
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
    for (int i = 0; i < n; i += U) {
        float v[U][VEC];
#pragma unroll
        for (int u = 0; u < U; ++u) load_vec<DT, VEC>(dy + (size_t)__builtin_amdgcn_readlane(pos, min(i + u, n - 1)) * a.N + at, v[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i + u >= n) break;
            const uint32_t k = __builtin_amdgcn_readlane(key, i + u);
            if (k != cur) {
                if (head)
                    partial(0);
                else
                    store();
                head = false;
                cur = k;
#pragma unroll
                for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] += v[u][e];
        }
    }
    if (head)
        partial(0);
    else if (next == cur)
        partial(1);
    else
        store();
}

// Joins the sums of the token that begins in a chunk and goes on after it, the chunk's own first. A wave per chunk and 64 VEC
// columns joins up to kFew following sums by itself, in order; longer runs (a token that is there hundreds of times) the block's
// waves join together, each every kFixWaves-th sum, and are added in order. A run of 1567 sums of 512 columns: 21 us (85 with
// loads that wait for one another), beside 13 for the sums of its 50160 rows.
constexpr int kFixWaves = 16, kFew = 16;
template <int DT, int VEC>
__global__ __launch_bounds__(64 * kFixWaves) void fixup_kernel(Sums a, void* __restrict__ dw_, int chunks) {
    using T = typename Row<DT>::T;
    constexpr int U = 16;
    const int part_of = blockIdx.x / a.slabs, slab = blockIdx.x - part_of * a.slabs;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = (slab * 64 + lane) * VEC;
    const bool mine = col < a.N;
    const float* part = a.part + (mine ? col : 0);
    T* dw = reinterpret_cast<T*>(dw_);
    __shared__ int ends[kFixWaves];  // the last chunk of a wave's run, for the block to join
    __shared__ uint32_t tokens[kFixWaves];
    __shared__ float join[kFixWaves][64 * VEC];
    auto sums_of = [&](float* v, int chunk, int which) {
        const float* at = part + ((size_t)chunk * 2 + which) * a.ld;
        if constexpr (VEC == 4) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(at);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = x[e];
        } else {
            v[0] = *at;
        }
    };
    // The sums of chunks j, j + step, ... up to last.
    auto sum = [&](float* acc, int j, int last, int step) {
        for (; j <= last; j += step * U) {
            float v[U][VEC];
#pragma unroll
            for (int u = 0; u < U; ++u) sums_of(v[u], min(j + u * step, last), 0);  // (all under way, whether they count or not)
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[u][e] = j + u * step <= last ? v[u][e] : 0.f;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < VEC; ++e) acc[e] += v[u][e];
        }
    };
    auto own = [&](float* acc, int c) { sums_of(acc, c, 1); };
    auto store = [&](const float* acc, uint32_t token) {
        if (mine) store_vec<DT, VEC>(dw + (size_t)token * a.N + col, acc, a.scale);
    };
    // Whether chunk c is the first of a run, its token and the run's last chunk.
    auto run = [&](int c, uint32_t& token, int& last) {
        if (c + 1 >= chunks) return false;
        const int lo = c * a.chunk;
        token = a.key[lo + a.chunk - 1];
        const uint32_t next = a.key[lo + a.chunk], first = a.key[lo], prev = lo > 0 ? a.key[lo - 1] : (uint32_t)a.V;
        if (token >= (uint32_t)a.V || next != token || (first == token && prev == token)) return false;
        last = c + 1;
        for (int end = chunks, round = 0; end - last > 1; ++round) {  // (the last one that begins with the token: in [last, end))
            const int step = round ? (end - last + 63) / 64 : 1;  // (most runs end within 64 chunks)
            const long long j = (long long)last + (long long)step * (lane + 1);
            const int found = __popcll(__ballot(j < end && a.key[j * a.chunk] == token));
            last += found * step;
            if (round || found < 64) end = min(end, last + step);
        }
        return true;
    };
    const int c = part_of * kFixWaves + wave;
    uint32_t token = 0;
    int last;
    int longer = 0;
    float acc[VEC];
    if (run(c, token, last)) {
        if (last - c <= kFew) {
            own(acc, c);
            sum(acc, c + 1, last, 1);
            store(acc, token);
        } else {
            longer = last;
        }
    }
    if (lane == 0) ends[wave] = longer, tokens[wave] = token;
    __syncthreads();
    for (int w = 0; w < kFixWaves; ++w) {
        if (ends[w] == 0) continue;
        const int c = part_of * kFixWaves + w;
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
        if (wave == 0) own(acc, c);
        sum(acc, c + 1 + wave, ends[w], kFixWaves);
#pragma unroll
        for (int e = 0; e < VEC; ++e) join[wave][lane * VEC + e] = acc[e];
        __syncthreads();
        if (wave == 0) {
#pragma unroll
            for (int v = 1; v < kFixWaves; ++v)
#pragma unroll
                for (int e = 0; e < VEC; ++e) acc[e] += join[v][lane * VEC + e];
            store(acc, tokens[w]);
        }
        __syncthreads();
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

size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }

struct Plan {
    int passes, nb, per, chunk, chunks, ld;
    size_t key[2], pos[2], counts, part, bytes;  // offsets into the workspace
    Plan(int64_t M, int64_t V, int64_t N) {
        passes = 1;
        while (((int64_t)1 << (passes * kDigit)) <= V) ++passes;  // keys 0 .. V
        per = (int)(std::max<int64_t>(1, (M + (int64_t)kMostSortBlocks * kSub - 1) / ((int64_t)kMostSortBlocks * kSub)) * kSub);
        nb = (int)((M + per - 1) / per);
        // Enough chunks for the chip, and chunks long enough that the borders' partial sums stay a small share.
        chunk = 8;
        while (chunk < 64 && M / chunk > 2048) chunk *= 2;
        chunks = (int)((M + chunk - 1) / chunk);
        ld = (int)((N + 3) & ~(int64_t)3);
        size_t n = 0;
        auto take = [&](size_t b) {
            const size_t at = n;
            n += up16(b);
            return at;
        };
        for (int i = 0; i < 2; ++i) key[i] = take(4 * (size_t)M), pos[i] = take(4 * (size_t)M);
        counts = take((size_t)nb * kBins * 4);
        part = take((size_t)chunks * 2 * ld * 4);
        bytes = n;
    }
};

bool sizes_ok(int64_t M, int64_t V, int64_t N) {
    return M >= 0 && M < ((int64_t)1 << 31) && V >= 1 && V < (1 << 27) && N >= 1 && N < (1 << 20) && V * N < ((int64_t)1 << 42) &&
           M * N < ((int64_t)1 << 42);
}
int check(int64_t M, int64_t V, int64_t N, int dtype, int idx_bits, const void* a, const void* b) {
    g_err.clear();
    if (!sizes_ok(M, V, N)) return fail("invalid sizes");
    if (dtype != kF16 && dtype != kBF16 && dtype != kF32) return fail("dtype must be float16, bfloat16 or float32");
    if (idx_bits != 32 && idx_bits != 64) return fail("tokens must be int32 or int64");
    if (((uintptr_t)a & 15) || ((uintptr_t)b & 15)) return fail("tensors must be 16-byte aligned");
    return 0;
}

template <typename F>
int by_dtype(int dtype, F f) {
    return dtype == kBF16 ? f(std::integral_constant<int, kBF16>()) : dtype == kF16 ? f(std::integral_constant<int, kF16>())
                                                                                    : f(std::integral_constant<int, kF32>());
}
template <typename F>
int by_index(int bits, F f) {
    return bits == 64 ? f((long long)0) : f((int)0);
}

}  // namespace

NNEMB_API const char* nn_embedding_last_error(void) { return g_err.c_str(); }

NNEMB_API int nn_embedding_fwd(const void* weight, const void* idx, void* out, int64_t M, int64_t V, int64_t N, float scale, int dtype,
                               int idx_bits, void* stream) {
    if (int e = check(M, V, N, dtype, idx_bits, weight, out)) return e;
    if (M == 0) return 0;
    if (!weight || !idx || !out) return fail("null pointer argument");
    return by_dtype(dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        return by_index(idx_bits, [&](auto i) {
            using I = decltype(i);
            auto go = [&](auto kern, int64_t per_row) {
                const int64_t units = M * per_row, blocks = (units + kThreads * kFwdUnits - 1) / (kThreads * kFwdUnits);
                if (blocks >= ((int64_t)1 << 32) / kThreads) return fail("invalid sizes");
                kern<<<dim3((unsigned)blocks), dim3(kThreads), 0, (hipStream_t)stream>>>(weight, (const I*)idx, out, units, (int)per_row, (int)V, scale);
                return launched("embedding fwd_kernel");
            };
            constexpr int W = Row<DT>::W;
            // What the next kernel can still find in the 256 MB cache is left there; half of it and more is stored past it.
            // With the norm that follows: 8192 x 768 fp32 (25 MB) 20 us, 22 past the caches; 131072 x 768 bf16 (201 MB) 139 us
            // either way, and the lookup itself 45 and 41 us (62 and 42 where other work has left the cache full).
            const bool past = M * N * (dtype == kF32 ? 4 : 2) >= (int64_t)128 << 20;
            return N % W     ? go(fwd_kernel<DT, 1, false, I>, N)
                   : past    ? go(fwd_kernel<DT, W, true, I>, N / W)
                             : go(fwd_kernel<DT, W, false, I>, N / W);
        });
    });
}

NNEMB_API size_t nn_embedding_bwd_workspace_size(int64_t M, int64_t V, int64_t N) {
    return sizes_ok(M, V, N) ? Plan(M, V, N).bytes : 0;
}

NNEMB_API int nn_embedding_bwd(const void* dy, const void* idx, void* dw, void* workspace, size_t workspace_bytes, int64_t M, int64_t V,
                               int64_t N, float scale, int64_t padding_idx, int dtype, int idx_bits, void* stream) {
    if (int e = check(M, V, N, dtype, idx_bits, dy, dw)) return e;
    const Plan p(M, V, N);
    if (workspace_bytes < p.bytes) return fail("workspace too small");
    if ((uintptr_t)workspace & 15) return fail("workspace must be 16-byte aligned");
    if (!dw || (M && (!dy || !idx || !workspace))) return fail("null pointer argument");
    const hipStream_t st = (hipStream_t)stream;
    const int64_t total = V * N * (dtype == kF32 ? 4 : 2), units = total / 16;
    constexpr int kFillBlocks = 1024, kSmallFill = 255;  // (one block to a CU where their LDS is the sort's)
    // The i-th of n launches' share of dW.
    auto share = [&](int i, int n) {
        return Fill{(u32x4*)dw, units * i / n, units * (i + 1) / n, (u16*)((char*)dw + units * 16), i + 1 == n ? (int)(total - units * 16) / 2 : 0};
    };
    if (M == 0) {
        fill_kernel<<<dim3(kFillBlocks), dim3(kSortThreads), 0, st>>>(share(0, 1));
        return launched("embedding fill_kernel");
    }
    char* ws = (char*)workspace;
    int* counts = (int*)(ws + p.counts);
    const bool small = M <= kSmall;
    if (small) {
        const int to = (p.passes - 1) & 1;
        const Pairs in{idx, nullptr, nullptr, padding_idx, (int)V, 0};
        const int e = by_index(idx_bits, [&](auto i) {
            sort_small_kernel<decltype(i)><<<dim3(1 + kSmallFill), dim3(kSmallThreads), 0, st>>>(in, (int)M, p.passes, (uint32_t*)(ws + p.key[to]),
                                                                                                 (int*)(ws + p.pos[to]), share(0, 1));
            return launched("embedding sort_small_kernel");
        });
        if (e) return e;
    }
    const int grid = p.nb + kFillBlocks, parts = 2 * p.passes;
    for (int pass = 0; pass < p.passes && !small; ++pass) {
        const int from = (pass + 1) & 1, to = pass & 1;
        const Pairs in{idx, (const uint32_t*)(ws + p.key[from]), (const int*)(ws + p.pos[from]), padding_idx, (int)V, pass * kDigit};
        uint32_t* key = (uint32_t*)(ws + p.key[to]);
        int* pos = (int*)(ws + p.pos[to]);
        const int e = by_index(idx_bits, [&](auto i) {
            using I = decltype(i);
            auto go = [&](auto count, auto place) {
                count<<<dim3(grid), dim3(kSortThreads), 0, st>>>(in, (int)M, p.per, p.nb, counts, share(2 * pass, parts));
                if (int err = launched("embedding count_kernel")) return err;
                place<<<dim3(grid), dim3(kSortThreads), 0, st>>>(in, (int)M, p.per, p.nb, counts, key, pos, share(2 * pass + 1, parts));
                return launched("embedding place_kernel");
            };
            return pass == 0 ? go(count_kernel<I, true>, place_kernel<I, true>) : go(count_kernel<I, false>, place_kernel<I, false>);
        });
        if (e) return e;
    }
    const int last = (p.passes - 1) & 1;
    return by_dtype(dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        auto go = [&](auto sum, auto fixup, int vec) {
            const int slabs = (int)((N + 64 * vec - 1) / (64 * vec));
            const int64_t waves = (int64_t)p.chunks * slabs, blocks = (waves + kThreads / 64 - 1) / (kThreads / 64);
            if (waves >= ((int64_t)1 << 32) / 64 - 64 * kFixWaves * slabs) return fail("invalid sizes");
            const Sums a{(const uint32_t*)(ws + p.key[last]), (const int*)(ws + p.pos[last]), (float*)(ws + p.part), (int)M, (int)V, (int)N,
                         p.ld, p.chunk, slabs, scale};
            sum<<<dim3((unsigned)blocks), dim3(kThreads), 0, st>>>(a, dy, dw, (long long)waves);
            if (int err = launched("embedding sum_kernel")) return err;
            if (p.chunks == 1) return 0;
            fixup<<<dim3((unsigned)((p.chunks + kFixWaves - 1) / kFixWaves * slabs)), dim3(64 * kFixWaves), 0, st>>>(a, dw, p.chunks);
            return launched("embedding fixup_kernel");
        };
        return N % 4 == 0 ? go(sum_kernel<DT, 4>, fixup_kernel<DT, 4>, 4) : go(sum_kernel<DT, 1>, fixup_kernel<DT, 1>, 1);
    });
}
