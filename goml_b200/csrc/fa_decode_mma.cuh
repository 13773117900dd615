// fa_decode_mma.cuh — warp-level products of decode attention, the conversions around them, and the sum of softmax states.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

namespace fa_sm100 {

// D = A B with a zero accumulator input
__device__ __forceinline__ void mma_e4m3_zero(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_f16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// four e4m3 bytes -> two fp16 pairs
__device__ __forceinline__ void e4m3_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
}

// One softmax state: maximum (log2 units), sum of weights and four columns of weighted values
struct State {
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    __device__ __forceinline__ void add(float m2, float l2, const float4& o2) {
        const float top = fmaxf(m, m2);
        if (top == -INFINITY) {   // nothing is seen, or nothing but NaNs
            l += l2;
            o.x += o2.x; o.y += o2.y; o.z += o2.z; o.w += o2.w;
            return;
        }
        const float f = exp2_fast(m - top), f2 = exp2_fast(m2 - top);
        m = top;
        l = l * f + l2 * f2;
        o.x = o.x * f + o2.x * f2; o.y = o.y * f + o2.y * f2; o.z = o.z * f + o2.z * f2; o.w = o.w * f + o2.w * f2;
    }
    // n states, eight of them on their way at a time; at(i): the place of the i-th
    template <int D, class At>
    __device__ __forceinline__ void add_all(const float* ml, const float* os, int n, int col, At&& at) {
        for (int i0 = 0; i0 < n; i0 += 8) {
            float2 x[8];
            float4 y[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                x[k] = make_float2(-INFINITY, 0.f);
                y[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (i0 + k >= n) continue;
                const size_t i = at(i0 + k);
                x[k] = __ldcg(reinterpret_cast<const float2*>(ml + 2 * i));
                y[k] = __ldcg(reinterpret_cast<const float4*>(os + i * D + col));
            }
            // against their common maximum: one state's factors do not wait for another's
            float top = m;
#pragma unroll
            for (int k = 0; k < 8; k++) top = fmaxf(top, x[k].x);
            const float base = top == -INFINITY ? 0.f : top, f = exp2_fast(m - base);   // nothing is seen, or nothing but NaNs: all factors are zero or a NaN's
            m = top;
            l *= f;
            o.x *= f; o.y *= f; o.z *= f; o.w *= f;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float fk = exp2_fast(x[k].x - base);
                l += x[k].y * fk;
                o.x += y[k].x * fk; o.y += y[k].y * fk; o.z += y[k].z * fk; o.w += y[k].w * fk;
            }
        }
    }
};

// four columns of a row of O, and with the first of them its LSE
template <int D>
__device__ __forceinline__ void store_output(__half* o, float* lse, size_t row, int col, const State& s, float vds) {
    const float inv = s.l > 0.f ? vds / s.l : s.l == 0.f ? 0.f : s.l;   // a NaN stays one
    __half* h = o + row * D + col;
    const uint32_t lo = half2_bits(s.o.x * inv, s.o.y * inv), hi = half2_bits(s.o.z * inv, s.o.w * inv);
    if ((reinterpret_cast<uintptr_t>(o) & 7) == 0) {   // o need only be 2-byte aligned
        *reinterpret_cast<uint2*>(h) = make_uint2(lo, hi);
    } else {
        uint16_t* w = reinterpret_cast<uint16_t*>(h);
        w[0] = (uint16_t)lo; w[1] = (uint16_t)(lo >> 16); w[2] = (uint16_t)hi; w[3] = (uint16_t)(hi >> 16);
    }
    if (col == 0 && lse) lse[row] = s.l == 0.f ? -INFINITY : (s.m + log2f(s.l)) * 0.6931471805599453f;
}

}  // namespace fa_sm100
