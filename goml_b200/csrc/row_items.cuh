// row_items.cuh — what the row-local kernels of libfp8block.so share: the decode of an item's index and wide loads of activations.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace sm100 {

// Division by a run-time constant as multiply-high + shift (numerators below 2^31): the item -> (row, column)
// decodes below would otherwise cost more instructions than the arithmetic they feed.
struct FastDiv {
    uint32_t d, mul, shr;
    FastDiv() : d(1), mul(0), shr(0) {}
    explicit FastDiv(uint32_t div) : d(div), mul(0), shr(0) {
        if (div > 1) {
            uint32_t lg = 0;
            while ((1ull << lg) < div) lg++;
            const uint32_t p = 31 + lg;
            mul = (uint32_t)(((1ull << p) + div - 1) / div);
            shr = p - 32;
        }
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return d == 1 ? n : __umulhi(n, mul) >> shr; }
    __device__ __forceinline__ void divmod(uint32_t n, uint32_t& q, uint32_t& r) const {
        q = div(n);
        r = n - q * d;
    }
};
// 256-bit global loads (sm_100): one instruction per 16 bf16 / 8 fp32 values, 32-byte aligned addresses.  Coherent ones:
// see one_cluster.cuh, and the residual stream is updated in place
struct U8 {
    uint32_t v[8];
};
__device__ __forceinline__ U8 ld256(const void* p) {
    U8 r;
    asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r.v[0]), "=r"(r.v[1]), "=r"(r.v[2]), "=r"(r.v[3]), "=r"(r.v[4]), "=r"(r.v[5]), "=r"(r.v[6]), "=r"(r.v[7])
                 : "l"(p)
                 : "memory");
    return r;
}
__device__ __forceinline__ void bf16x16_to_f32(const U8& r, float* f) {
#pragma unroll
    for (int k = 0; k < 8; k++) {
        f[2 * k] = __uint_as_float(r.v[k] << 16);
        f[2 * k + 1] = __uint_as_float(r.v[k] & 0xffff0000u);
    }
}
__device__ __forceinline__ void bf16x8_to_f32(const uint4 v, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; k++) {
        f[2 * k] = __uint_as_float(w[k] << 16);
        f[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
    }
}

}  // namespace sm100
