// RMS norm of each query and key head's vector and its rotation by the token's position, in one pass, forward and backward,
// for MI355X (gfx950).
//
// Forward, for a vector x of D values: r = 1 / sqrt(mean(x^2) + eps), v = w (r x), y = R v with R the rotation of the pairs
// (i, i + D/2) by the position's angles. Backward, with g = R^T dy (the rotation back) and n = r x:
//     dw = sum over tokens and heads of g n,    dx = r (w g - n mean(w g n))
// r is computed again from x, which the backward reads anyway. Everything is fp32; an output is rounded once.
//
// Work decomposition. A vector belongs to a team of R lanes (R the power of two at or above D/16); a lane holds 8 pairs: two
// groups of 8 values. Sums over a vector are xor-butterflies over the team. The kernels are bound by memory.
//
// Forward: a team takes two heads of one token, queries or keys, which share the token's angles and the weight, whose fp32 values
// are twice as many bytes as a head's 16-bit ones and come from the caches (131072 tokens of 12 + 4 heads of 64 in bf16: 109 us,
// 4.9 TB/s; one head 113, four 115).
//
// Backward: a fixed grid whose blocks work on queries or on keys, in proportion; every team walks its kind's vectors and keeps
// its lanes' part of dw in registers. A block's teams are joined by butterflies within the waves and in LDS in wave order, into
// one partial row per block; sum_kernel adds a kind's rows in a fixed order: no atomics, bit-reproducible. 1024 blocks are what
// the chip holds at once (the same tokens: 165 us, 4.9 TB/s with the sums' 5; 768 blocks 172, 1280 222, 2048 173; two heads of
// a token at a time 174 to 203, four 178).
#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include <algorithm>
#include <string>

#include "nanonemo_qk_norm.h"
#include "rows.h"

#define NNQK_API extern "C" __attribute__((visibility("default")))

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kBwdBlocks = 1024;  // most blocks of the backward, each of which leaves one partial row of dw
constexpr int kFwdHeads = 2;      // heads of a token to a team of the forward
constexpr int kSumWaves = 16;

// 8 values of a row as fp32, and back.
template <int DT>
__device__ inline void load8(const char* base, long long at, float* v) {
    using R = Row<DT>;
    const typename R::T* p = reinterpret_cast<const typename R::T*>(base) + at;
    R::load(p, v);
    if constexpr (DT == kF32) R::load(p + 4, v + 4);
}
template <int DT>
__device__ inline void store8(char* base, long long at, const float* v) {
    using R = Row<DT>;
    typename R::T* p = reinterpret_cast<typename R::T*>(base) + at;
    R::store(p, v);
    if constexpr (DT == kF32) R::store(p + 4, v + 4);
}
__device__ inline void load8f(const float* p, float* v) { load8<kF32>(reinterpret_cast<const char*>(p), 0, v); }

struct Side {  // queries or keys
    const char* x;
    const char* dy;  // backward
    char* y;         // forward: the output; backward: dx
    const float* w;
    long long xt, xh, dt, dh, yt, yh;  // element strides {token, head} of x, dy and y
    int heads;
};
struct Angles {
    const float *cosT, *sinT;
    const void* positions;
    long long rows;
    unsigned period;
    int bits;
};

// The token's angles for pairs i0 .. i0 + 7; whether its position is a row of the tables (otherwise they are row 0's, and the
// callers make NaN of what they compute).
__device__ inline bool angles(const Angles& a, unsigned token, int half, int i0, float* c, float* s) {
    const unsigned m = token % a.period;
    const long long p = !a.positions ? m : a.bits == 64 ? static_cast<const long long*>(a.positions)[m] : static_cast<const int*>(a.positions)[m];
    const bool ok = p >= 0 && p < a.rows;
    const long long at = (ok ? p : 0) * half + i0;
    load8f(a.cosT + at, c);
    load8f(a.sinT + at, s);
    return ok;
}

template <int R>
__device__ inline float team_sum(float v) {
#pragma unroll
    for (int m = R / 2; m > 0; m >>= 1) v += __shfl_xor(v, m);
    return v;
}

// Blocks [0, qblocks) take the queries' units (NH heads of a token), the others the keys'.
template <int DT, int R, int NH>
__global__ __launch_bounds__(kThreads) void qk_norm_fwd_kernel(Side q, Side k, Angles a, unsigned tokens, unsigned qblocks, int D, float inv_d, float eps) {
    const int half = D / 2, lane = threadIdx.x % R, i0 = 8 * lane;
    const bool isq = blockIdx.x < qblocks;
    const int heads = isq ? q.heads : k.heads;
    const unsigned per = (heads + NH - 1) / NH, u = (isq ? blockIdx.x : blockIdx.x - qblocks) * (kThreads / R) + threadIdx.x / R;
    const unsigned token = u / per;
    if (token >= tokens) return;  // (whole teams)
    const int h0 = (int)(u - token * per) * NH;
    const char* x = isq ? q.x : k.x;
    char* y = isq ? q.y : k.y;
    const float* w = isq ? q.w : k.w;
    const long long xh = isq ? q.xh : k.xh, yh = isq ? q.yh : k.yh;
    const long long xo = token * (isq ? q.xt : k.xt) + h0 * xh + i0, yo = token * (isq ? q.yt : k.yt) + h0 * yh + i0;
    const bool on = i0 < half;
    float x1[NH][8], x2[NH][8], w1[8], w2[8], c[8], s[8];
#pragma unroll
    for (int n = 0; n < NH; ++n) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x1[n][j] = x2[n][j] = 0.f;
        if (on && h0 + n < heads) {
            load8<DT>(x, xo + n * xh, x1[n]);
            load8<DT>(x, xo + n * xh + half, x2[n]);
        }
    }
    bool ok = true;
    if (on) {
        ok = angles(a, token, half, i0, c, s);
        load8f(w + i0, w1);
        load8f(w + half + i0, w2);
    }
#pragma unroll
    for (int n = 0; n < NH; ++n) {
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(x1[n][j], x1[n][j], fmaf(x2[n][j], x2[n][j], ss));
        const float r = ok ? rsqrtf(team_sum<R>(ss) * inv_d + eps) : NAN;
        if (!on || h0 + n >= heads) continue;
        float y1[8], y2[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float v1 = x1[n][j] * r * w1[j], v2 = x2[n][j] * r * w2[j];
            y1[j] = v1 * c[j] - v2 * s[j];
            y2[j] = v1 * s[j] + v2 * c[j];
        }
        store8<DT>(y, yo + n * yh, y1);
        store8<DT>(y, yo + n * yh + half, y2);
    }
}

// Blocks [0, qblocks) take the queries' vectors, the others the keys'.
template <int DT, int R>
__global__ __launch_bounds__(kThreads) void qk_norm_bwd_kernel(Side q, Side k, Angles a, unsigned tokens, unsigned qblocks, float* __restrict__ part,
                                                               int D, float inv_d, float eps) {
    __shared__ float red[kWaves][16 * 16];
    const int half = D / 2, lane = threadIdx.x % R, i0 = 8 * lane;
    const bool isq = blockIdx.x < qblocks, on = i0 < half;
    const unsigned blocks = isq ? qblocks : gridDim.x - qblocks, block = isq ? blockIdx.x : blockIdx.x - qblocks;
    const char* x = isq ? q.x : k.x;
    const char* dy = isq ? q.dy : k.dy;
    char* dx = isq ? q.y : k.y;
    const float* w = isq ? q.w : k.w;
    const long long xt = isq ? q.xt : k.xt, xh = isq ? q.xh : k.xh, dt = isq ? q.dt : k.dt, dh = isq ? q.dh : k.dh, yt = isq ? q.yt : k.yt,
                    yh = isq ? q.yh : k.yh;
    const unsigned heads = isq ? q.heads : k.heads, vectors = tokens * heads, teams = blocks * (kThreads / R);
    float w1[8] = {}, w2[8] = {}, a1[8] = {}, a2[8] = {};
    if (on) {
        load8f(w + i0, w1);
        load8f(w + half + i0, w2);
    }
    for (unsigned u = block * (kThreads / R) + threadIdx.x / R; u < vectors; u += teams) {
        const unsigned token = u / heads, h = u - token * heads;
        float x1[8] = {}, x2[8] = {}, g1[8] = {}, g2[8] = {};
        bool ok = true;
        if (on) {
            const long long xo = token * xt + h * xh + i0, go = token * dt + h * dh + i0;
            float d1[8], d2[8], c[8], s[8];
            load8<DT>(x, xo, x1);
            load8<DT>(x, xo + half, x2);
            load8<DT>(dy, go, d1);
            load8<DT>(dy, go + half, d2);
            ok = angles(a, token, half, i0, c, s);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                g1[j] = d1[j] * c[j] + d2[j] * s[j];
                g2[j] = d2[j] * c[j] - d1[j] * s[j];
            }
        }
        float ss = 0.f, gx = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            ss = fmaf(x1[j], x1[j], fmaf(x2[j], x2[j], ss));
            gx = fmaf(g1[j] * w1[j], x1[j], fmaf(g2[j] * w2[j], x2[j], gx));
        }
        const float r = ok ? rsqrtf(team_sum<R>(ss) * inv_d + eps) : NAN, m = r * team_sum<R>(gx) * inv_d;
        if (!on) continue;
        float y1[8], y2[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float n1 = x1[j] * r, n2 = x2[j] * r;
            a1[j] = fmaf(g1[j], n1, a1[j]);
            a2[j] = fmaf(g2[j], n2, a2[j]);
            y1[j] = r * (g1[j] * w1[j] - n1 * m);
            y2[j] = r * (g2[j] * w2[j] - n2 * m);
        }
        const long long yo = token * yt + h * yh + i0;
        store8<DT>(dx, yo, y1);
        store8<DT>(dx, yo + half, y2);
    }
    // The wave's teams, then the block's waves.
#pragma unroll
    for (int m = R; m < 64; m <<= 1)
#pragma unroll
        for (int j = 0; j < 8; ++j) a1[j] += __shfl_xor(a1[j], m), a2[j] += __shfl_xor(a2[j], m);
    const int wave = threadIdx.x / 64;
    if (threadIdx.x % 64 < R && on) {
#pragma unroll
        for (int j = 0; j < 8; ++j) red[wave][i0 + j] = a1[j], red[wave][half + i0 + j] = a2[j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < D; i += kThreads) {
        float v = red[0][i];
#pragma unroll
        for (int n = 1; n < kWaves; ++n) v += red[n][i];
        part[(size_t)blockIdx.x * D + i] = v;
    }
}

// dw of queries (blockIdx.y 0: rows [0, qrows) of part) or keys (the rows after them): a wave adds every 16th row of 64 columns,
// then the waves' sums in order.
__global__ __launch_bounds__(64 * kSumWaves) void qk_norm_sum_kernel(const float* __restrict__ part, int qrows, int rows, int D, float* __restrict__ dwq,
                                                                     float* __restrict__ dwk) {
    __shared__ float red[kSumWaves][64];
    const int col = blockIdx.x * 64 + threadIdx.x % 64, wave = threadIdx.x / 64;
    const int from = blockIdx.y ? qrows : 0, to = blockIdx.y ? rows : qrows;
    float v = 0.f;
    if (col < D) {
#pragma unroll 8
        for (int r = from + wave; r < to; r += kSumWaves) v += part[(size_t)r * D + col];
    }
    red[wave][threadIdx.x % 64] = v;
    __syncthreads();
    if (wave || col >= D) return;
#pragma unroll
    for (int n = 1; n < kSumWaves; ++n) v += red[n][threadIdx.x];
    (blockIdx.y ? dwk : dwq)[col] = v;
}

thread_local std::string g_err;
int fail(const char* fmt, ...) __attribute__((format(printf, 1, 2)));
int fail(const char* fmt, ...) {
    char buf[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    g_err = buf;
    return -1;
}
int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return 0;
    fail("%s launch failed: %s", what, hipGetErrorString(e));
    return (int)e;
}
bool aligned(const void* p, int n) { return ((uintptr_t)p % n) == 0; }

// Lanes per vector.
int team_of(int64_t D) {
    int r = 1;
    while (r * 16 < D) r *= 2;
    return r;
}

// Blocks on queries and on keys, with a team for each unit of NH heads.
struct Grid {
    unsigned q, k;
};
Grid grid_of(int64_t M, int64_t H, int64_t KVH, int64_t D, int NH) {
    const int64_t teams = kThreads / team_of(D);
    const int64_t qu = M * ((H + NH - 1) / NH), ku = M * ((KVH + NH - 1) / NH);
    return {(unsigned)((qu + teams - 1) / teams), (unsigned)((ku + teams - 1) / teams)};
}
// The backward's: kBwdBlocks at most, in proportion to the heads.
Grid bwd_grid(int64_t M, int64_t H, int64_t KVH, int64_t D) {
    if (M <= 0) return {0, 0};
    const Grid all = grid_of(M, H, KVH, D, 1);
    const int64_t qb = all.q, kb = all.k;
    if (qb + kb <= kBwdBlocks) return all;
    const int64_t q = std::min<int64_t>(kBwdBlocks - 1, std::max<int64_t>(1, (kBwdBlocks * H + (H + KVH) / 2) / (H + KVH)));
    return {(unsigned)std::min(q, qb), (unsigned)std::min(kBwdBlocks - q, kb)};
}

int check(int64_t M, int64_t H, int64_t KVH, int64_t D, int dtype, const int64_t* strides, int nstrides, const float* wq, const float* wk,
          const float* cos_table, const float* sin_table, int64_t table_rows, const void* positions, int bits, int64_t period) {
    g_err.clear();
    if (M < 0 || H <= 0 || KVH <= 0 || table_rows < 0) return fail("invalid sizes");
    if (D <= 0 || D % 16 || D > 256) return fail("head_dim must be a multiple of 16, up to 256");
    if (dtype != kF16 && dtype != kBF16 && dtype != kF32) return fail("dtype must be float16, bfloat16 or float32");
    if (!strides) return fail("null strides");
    for (int i = 0; i < nstrides; ++i)
        if (strides[i] <= 0 || strides[i] % 8 || strides[i] >= (int64_t)1 << 40) return fail("strides must be positive multiples of 8 elements");
    // (a launch's threads, and a unit's 32-bit index with a grid's more than the last)
    if (M >= (int64_t)1 << 31 || H >= (int64_t)1 << 31 || KVH >= (int64_t)1 << 31 || M * (H + KVH) >= ((int64_t)1 << 31) / team_of(D))
        return fail("sizes too large");
    if (M == 0) return 0;
    if (!wq || !wk || !cos_table || !sin_table) return fail("null weight or table");
    if (!aligned(wq, 16) || !aligned(wk, 16) || !aligned(cos_table, 16) || !aligned(sin_table, 16)) return fail("weights and tables must be 16-byte aligned");
    if (table_rows == 0) return fail("the tables have no rows");
    if (period <= 0 || period >= (int64_t)1 << 31) return fail("invalid period");
    if (positions) {
        if (bits != 32 && bits != 64) return fail("positions must be int32 or int64");
        if (!aligned(positions, bits / 8)) return fail("positions must be aligned");
    } else if (std::min(M, period) > table_rows) {
        return fail("sequence length %lld exceeds the %lld rows of the tables", (long long)std::min(M, period), (long long)table_rows);
    }
    return 0;
}

// One of the kernels for R lanes per vector.
template <class F>
int with_team(int R, F f) {
    switch (R) {
        case 1: return f(std::integral_constant<int, 1>{});
        case 2: return f(std::integral_constant<int, 2>{});
        case 4: return f(std::integral_constant<int, 4>{});
        case 8: return f(std::integral_constant<int, 8>{});
        default: return f(std::integral_constant<int, 16>{});
    }
}
template <class F>
int with_type(int dtype, F f) {
    return dtype == kBF16 ? f(std::integral_constant<int, kBF16>{}) : dtype == kF16 ? f(std::integral_constant<int, kF16>{}) : f(std::integral_constant<int, kF32>{});
}

}  // namespace

NNQK_API const char* nn_qk_norm_last_error(void) { return g_err.c_str(); }

NNQK_API int nn_qk_norm_rope_fwd(const void* q, const void* k, const float* q_weight, const float* k_weight, const float* cos_table,
                                 const float* sin_table, int64_t table_rows, const void* positions, int position_bits, int64_t period,
                                 void* q_out, void* k_out, int64_t M, int64_t H, int64_t KVH, int64_t D, const int64_t* strides, float eps, int dtype,
                                 void* stream) {
    if (int e = check(M, H, KVH, D, dtype, strides, 8, q_weight, k_weight, cos_table, sin_table, table_rows, positions, position_bits, period)) return e;
    if (M == 0) return 0;
    if (!q || !k || !q_out || !k_out) return fail("null pointer argument");
    if (!aligned(q, 16) || !aligned(k, 16) || !aligned(q_out, 16) || !aligned(k_out, 16)) return fail("tensors must be 16-byte aligned");
    const Side qs{(const char*)q, nullptr, (char*)q_out, q_weight, strides[0], strides[1], 0, 0, strides[4], strides[5], (int)H};
    const Side ks{(const char*)k, nullptr, (char*)k_out, k_weight, strides[2], strides[3], 0, 0, strides[6], strides[7], (int)KVH};
    const Angles a{cos_table, sin_table, positions, table_rows, (unsigned)period, position_bits};
    const Grid g = grid_of(M, H, KVH, D, kFwdHeads);
    return with_type(dtype, [&](auto dt) {
        return with_team(team_of(D), [&](auto r) {
            qk_norm_fwd_kernel<dt(), r(), kFwdHeads><<<dim3(g.q + g.k), dim3(kThreads), 0, (hipStream_t)stream>>>(qs, ks, a, (unsigned)M, g.q, (int)D,
                                                                                                              1.f / (float)D, eps);
            return launched("qk_norm_fwd_kernel");
        });
    });
}

NNQK_API size_t nn_qk_norm_rope_bwd_workspace_size(int64_t M, int64_t H, int64_t KVH, int64_t D) {
    if (M <= 0 || H <= 0 || KVH <= 0 || D <= 0 || D > 256 || M >= (int64_t)1 << 31 || H >= (int64_t)1 << 31 || KVH >= (int64_t)1 << 31) return 0;
    const Grid g = bwd_grid(M, H, KVH, D);
    return (size_t)(g.q + g.k) * D * 4;
}

NNQK_API int nn_qk_norm_rope_bwd(const void* dq_out, const void* dk_out, const void* q, const void* k, const float* q_weight, const float* k_weight,
                                 const float* cos_table, const float* sin_table, int64_t table_rows, const void* positions, int position_bits,
                                 int64_t period, void* dq, void* dk, float* dq_weight, float* dk_weight, void* workspace, size_t workspace_bytes,
                                 int64_t M, int64_t H, int64_t KVH, int64_t D, const int64_t* strides, float eps, int dtype, void* stream) {
    if (int e = check(M, H, KVH, D, dtype, strides, 12, q_weight, k_weight, cos_table, sin_table, table_rows, positions, position_bits, period)) return e;
    if (!dq_weight || !dk_weight) return fail("null pointer argument");
    const Grid g = bwd_grid(M, H, KVH, D);
    const hipStream_t st = (hipStream_t)stream;
    if (M > 0) {
        if (!dq_out || !dk_out || !q || !k || !dq || !dk) return fail("null pointer argument");
        for (const void* p : {dq_out, dk_out, q, k, (const void*)dq, (const void*)dk})
            if (!aligned(p, 16)) return fail("tensors must be 16-byte aligned");
        const size_t need = (size_t)(g.q + g.k) * D * 4;
        if (!workspace || !aligned(workspace, 16) || workspace_bytes < need) return fail("workspace of %zu bytes needed, 16-byte aligned", need);
        const Side qs{(const char*)q, (const char*)dq_out, (char*)dq, q_weight, strides[4], strides[5], strides[0], strides[1], strides[8], strides[9], (int)H};
        const Side ks{(const char*)k, (const char*)dk_out, (char*)dk, k_weight, strides[6], strides[7], strides[2], strides[3], strides[10], strides[11], (int)KVH};
        const Angles a{cos_table, sin_table, positions, table_rows, (unsigned)period, position_bits};
        const int e = with_type(dtype, [&](auto dt) {
            return with_team(team_of(D), [&](auto r) {
                qk_norm_bwd_kernel<dt(), r()><<<dim3(g.q + g.k), dim3(kThreads), 0, st>>>(qs, ks, a, (unsigned)M, g.q, (float*)workspace, (int)D,
                                                                                                          1.f / (float)D, eps);
                return launched("qk_norm_bwd_kernel");
            });
        });
        if (e) return e;
    }
    qk_norm_sum_kernel<<<dim3((unsigned)((D + 63) / 64), 2), dim3(64 * kSumWaves), 0, st>>>((const float*)workspace, (int)g.q, (int)(g.q + g.k), (int)D,
                                                                                          dq_weight, dk_weight);
    return launched("qk_norm_sum_kernel");
}
