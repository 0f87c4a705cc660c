// Rows of fp16, bf16 or fp32 values read and written in 16-byte groups as fp32, for the row kernels of MI355X (gfx950)
// (losses, top logits, embedding).
#pragma once
#include <type_traits>

#include "tiles.h"

namespace {

constexpr int kF32 = 2;

// Values of type DT in groups of 16 bytes, as fp32.
template <int DT>
struct Row {
    static constexpr int W = DT == kF32 ? 4 : 8;
    using T = std::conditional_t<DT == kF32, float, u16>;
    static __device__ float one(T x) {
        if constexpr (DT == kF32)
            return x;
        else
            return Elem<DT>::to_f32(x);
    }
    static __device__ T round(float x) {
        if constexpr (DT == kF32)
            return x;
        else
            return (T)(Elem<DT>::pack2(x, 0.f) & 0xffffu);
    }
    // A group's 16 bytes as fp32, and back.
    static __device__ void widen(u32x4 raw, float* v) {
        if constexpr (DT == kF32) {
            const f32x4 x = __builtin_bit_cast(f32x4, raw);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = x[e];
        } else {
            const u16x8 x = __builtin_bit_cast(u16x8, raw);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = Elem<DT>::to_f32(x[e]);
        }
    }
    static __device__ u32x4 narrow(const float* v) {
        if constexpr (DT == kF32)
            return __builtin_bit_cast(u32x4, f32x4{v[0], v[1], v[2], v[3]});
        else
            return u32x4{Elem<DT>::pack2(v[0], v[1]), Elem<DT>::pack2(v[2], v[3]), Elem<DT>::pack2(v[4], v[5]), Elem<DT>::pack2(v[6], v[7])};
    }
    static __device__ u32x4 raw(const T* p) { return *reinterpret_cast<const u32x4*>(p); }
    static __device__ void load(const T* p, float* v) { widen(raw(p), v); }
    static __device__ void store(T* p, const float* v) { *reinterpret_cast<u32x4*>(p) = narrow(v); }
    // Values before the row's first 16-byte boundary (rows of an odd vocabulary start anywhere).
    static __device__ int head(const T* row, int V) { return min(V, (int)((16 - ((uintptr_t)row & 15)) & 15) / (int)sizeof(T)); }
};

}  // namespace
