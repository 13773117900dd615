// fp4_cache_sm100.cu — rows into and out of a KV cache held in 4 bits (fp4_rope_append and fp4_cache_rows, include/fp8_block.h).
//
// Both are one pass over their rows, a thread to 32 dims of one (token, head): RoPE pairs dim i with dim i + hd/2, so a thread that takes 16 dims of one half and
// their partners of the other has two whole groups of 16, whose scales it finds by itself.  HBM-bound: an append reads 2 bytes a value of the projection
// and writes 2 of the queries and 0.56 of keys and values.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/fp8_block.h"
#include "pdl.cuh"
#include "row_items.cuh"

namespace {

using namespace sm100;

constexpr int THREADS = 256;
constexpr int CTAS_PER_SM = 8;

int grid_for(size_t items) {
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    const size_t blocks = (items + THREADS - 1) / THREADS, cap = (size_t)sms * CTAS_PER_SM;
    return (int)(blocks < cap ? blocks : cap);
}
bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// A number near a float q whose last KEEP bits of 23 are zero, if q lies within a few units in the last place of one: the places where the rounding of a
// quotient could hide on which side of a border between two codes it lies
template <int DROP>
__device__ __forceinline__ bool near_short(uint32_t q, uint32_t& at) {
    at = (q + (1u << (DROP - 1))) & ~((1u << DROP) - 1u);
    return q - at + 8u <= 16u;
}
__device__ __forceinline__ uint32_t nudged(uint32_t at, float residual) { return at + (residual > 0.f ? 1u : 0u) - (residual < 0.f ? 1u : 0u); }

// A tensor scale and what the quotients by it need
struct TensorScale {
    float s, six, six_rest, inv_six;   // six + six_rest is 6 s exactly
    __device__ __forceinline__ explicit TensorScale(float scale) : s(scale) {
        six = __fmul_rn(6.f, s);
        six_rest = __fmaf_rn(6.f, s, -six);
        inv_six = __fdiv_rn(1.f, six);
    }
};

// e4m3(a / 6s), a >= 0 given by its bits.  Borders between e4m3 numbers have at most five significant bits.
__device__ __forceinline__ uint32_t block_scale(uint32_t a_bits, const TensorScale& ts) {
    const float a = __uint_as_float(a_bits);
    uint32_t q = __float_as_uint(__fmul_rn(a, ts.inv_six)), at;
    if (near_short<19>(q, at)) {
        const float m = __uint_as_float(at);
        q = nudged(at, __fmaf_rn(-m, ts.six_rest, __fmaf_rn(-m, ts.six, a)));   // the first is exact: a and m * six cancel to their last bits
    }
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(__uint_as_float(q)));
    return r & 0xffu;
}
__device__ __forceinline__ float e4m3_to_f32(uint32_t b) {
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(r) : "r"(b));
    return __half2float(__low2half(*reinterpret_cast<const __half2*>(&r)));
}
// y / d as a number that rounds to the code that the exact quotient rounds to.  Borders between codes have at most three significant bits; the residual of one is
// exact in its sign.
__device__ __forceinline__ float code_quotient(float y, float d, float inv) {
    const uint32_t sign = __float_as_uint(y) & 0x80000000u;
    const float a = fabsf(y);
    uint32_t q = __float_as_uint(__fmul_rn(a, inv)), at;
    if (near_short<21>(q, at)) q = nudged(at, __fmaf_rn(-__uint_as_float(at), d, a));
    return __uint_as_float(q | sign);
}
// A group of 16 values: its codes, and its block scale as the result
__device__ __forceinline__ uint32_t quantise16(const float* y, const TensorScale& ts, uint2& codes) {
    uint32_t top = 0;   // of the bits: a NaN is above every number
#pragma unroll
    for (int i = 0; i < 16; i++) top = max(top, __float_as_uint(y[i]) & 0x7fffffffu);
    codes = make_uint2(0u, 0u);
    if (top > 0x7f800000u) return 0x7fu;
    const uint32_t b = block_scale(top, ts);
    const float d = __fmul_rn(e4m3_to_f32(b), ts.s);
    if (d < 1.1754943508222875e-38f) return b;
    const float inv = __fdiv_rn(1.f, d);
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        float q[8];
#pragma unroll
        for (int i = 0; i < 8; i++) q[i] = code_quotient(y[8 * h + i], d, inv);
        asm("{\n\t.reg .b8 a, b, c, d;\n\tcvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
            "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\tmov.b32 %0, {a, b, c, d};\n\t}"
            : "=r"(w[h])
            : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]), "f"(q[4]), "f"(q[5]), "f"(q[6]), "f"(q[7]));
    }
    codes = make_uint2(w[0], w[1]);
    return b;
}

// What lies where in the cache: row = (page * kv_heads + head) * page_size + place
struct Cache {
    uint8_t *k, *ks, *v, *vs;
    const float *k_scale, *v_scale;
    int kv_heads, hd, page_size;
    uint32_t slots;   // num_pages * page_size
    FastDiv page;
    __device__ __forceinline__ size_t row(int slot, int head) const {
        uint32_t pg, place;
        page.divmod((uint32_t)slot, pg, place);
        return ((size_t)pg * kv_heads + head) * page_size + place;
    }
    __device__ __forceinline__ uint8_t* k_scale_at(size_t row, int group) const { return ks + row * (hd / 16) + group; }
    __device__ __forceinline__ uint8_t* v_scale_at(size_t row, int group) const { return vs + row / 16 * hd + group * 16 + row % 16; }
};

struct Append {
    const uint16_t* qkv;
    const float *cos_tab, *sin_tab;
    const int32_t *positions, *slots;
    uint16_t* q_out;
    Cache cache;
    uint32_t items;   // tokens * heads of a row * hd / 32
    int q_heads, rope_rows;
    FastDiv cph, heads;   // 32-dim pieces of a head, heads of a row
};
__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ void store_bf16x16(uint16_t* to, const float* y) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; i++) w[i] = bf16x2(y[2 * i], y[2 * i + 1]);
    reinterpret_cast<uint4*>(to)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    reinterpret_cast<uint4*>(to)[1] = make_uint4(w[4], w[5], w[6], w[7]);
}
__device__ __forceinline__ void load_bf16x16(const uint16_t* from, float* y) {
    bf16x8_to_f32(ld128(from), y);
    bf16x8_to_f32(ld128(from + 8), y + 8);
}

__global__ void __launch_bounds__(THREADS) fp4_append_kernel(const Append a) {
    pdl_wait();
    pdl_trigger();
    const int hd = a.cache.hd, half = hd / 2, kv = a.cache.kv_heads;
    for (uint32_t it = blockIdx.x * THREADS + threadIdx.x; it < a.items; it += gridDim.x * THREADS) {
        uint32_t r, c, token, head;
        a.cph.divmod(it, r, c);
        a.heads.divmod(r, token, head);
        const bool is_q = (int)head < a.q_heads, is_v = (int)head >= a.q_heads + kv;
        const int pos = ld_s32(a.positions + token), slot = ld_s32(a.slots + token);
        const bool active = pos >= 0 && pos < a.rope_rows;
        if (is_q ? a.q_out == nullptr : !active || slot < 0 || (uint32_t)slot >= a.cache.slots) continue;
        // two groups of 16 dims: the two halves' c-th, of values the 2c-th and the one after it
        const int d0 = is_v ? 32 * c : 16 * c, d1 = is_v ? 32 * c + 16 : half + 16 * c;
        float y[32];
        if (active) {
            const uint16_t* x = a.qkv + (size_t)r * hd;
            load_bf16x16(x + d0, y);
            load_bf16x16(x + d1, y + 16);
            if (!is_v) {
                const float* cs = a.cos_tab + (size_t)pos * half + 16 * c;
                const float* sn = a.sin_tab + (size_t)pos * half + 16 * c;
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const float cc = ld_f32(cs + i), ss = ld_f32(sn + i), x0 = y[i], x1 = y[16 + i];
                    y[i] = __fsub_rn(__fmul_rn(x0, cc), __fmul_rn(x1, ss));
                    y[16 + i] = __fadd_rn(__fmul_rn(x0, ss), __fmul_rn(x1, cc));
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 32; i++) y[i] = 0.f;
        }
        if (is_q) {
            uint16_t* q = a.q_out + ((size_t)token * a.q_heads + head) * hd;
            store_bf16x16(q + d0, y);
            store_bf16x16(q + d1, y + 16);
            continue;
        }
        const int h = (int)head - a.q_heads - (is_v ? kv : 0);
        const size_t row = a.cache.row(slot, h);
        const TensorScale ts(ld_f32(is_v ? a.cache.v_scale : a.cache.k_scale));
        uint8_t* codes = (is_v ? a.cache.v : a.cache.k) + row * half;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int d = j ? d1 : d0;
            uint2 w;
            const uint32_t b = quantise16(y + 16 * j, ts, w);
            *reinterpret_cast<uint2*>(codes + d / 2) = w;
            *(is_v ? a.cache.v_scale_at(row, d / 16) : a.cache.k_scale_at(row, d / 16)) = (uint8_t)b;
        }
    }
}

struct Rows {
    const int32_t* slots;
    uint16_t *k_out, *v_out;
    Cache cache;
    uint32_t items;   // tokens * kv heads * hd / 16, of keys and then as many of values
    FastDiv groups, heads;
};
__global__ void __launch_bounds__(THREADS) fp4_rows_kernel(const Rows a) {
    pdl_wait();
    pdl_trigger();
    const int hd = a.cache.hd;
    for (uint32_t i = blockIdx.x * THREADS + threadIdx.x; i < 2 * a.items; i += gridDim.x * THREADS) {
        const bool is_v = i >= a.items;
        const uint32_t it = is_v ? i - a.items : i;
        uint32_t r, group, token, head;
        a.groups.divmod(it, r, group);
        a.heads.divmod(r, token, head);
        const int slot = ld_s32(a.slots + token);
        float y[16];
        if (slot >= 0 && (uint32_t)slot < a.cache.slots) {
            const size_t row = a.cache.row(slot, (int)head);
            const uint8_t* codes = (is_v ? a.cache.v : a.cache.k) + row * (hd / 2) + 8 * group;
            uint32_t w[2];
            asm volatile("ld.global.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(codes) : "memory");
            uint16_t b;
            asm volatile("ld.global.u8 %0, [%1];" : "=h"(b) : "l"(is_v ? a.cache.v_scale_at(row, group) : a.cache.k_scale_at(row, group)) : "memory");
            const float s = ld_f32(is_v ? a.cache.v_scale : a.cache.k_scale), bs = e4m3_to_f32(b);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                uint32_t x[4];
                asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
                    "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
                    : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                    : "r"(w[h]));
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x[j]));
                    y[8 * h + 2 * j] = __fmul_rn(__fmul_rn(f.x, bs), s);   // the first product is exact
                    y[8 * h + 2 * j + 1] = __fmul_rn(__fmul_rn(f.y, bs), s);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 16; j++) y[j] = 0.f;
        }
        store_bf16x16((is_v ? a.v_out : a.k_out) + (size_t)it * 16, y);
    }
}

bool cache_of(Cache& c, const void* k, const void* ks, const void* v, const void* vs, const float* k_scale, const float* v_scale, int kv_heads, int hd, int page_size,
              int num_pages) {
    if (!k || !ks || !v || !vs || !k_scale || !v_scale || !aligned(k, 16) || !aligned(ks, 16) || !aligned(v, 16) || !aligned(vs, 16) || !aligned(k_scale, 4) || !aligned(v_scale, 4))
        return false;
    if (kv_heads <= 0 || (hd != 64 && hd != 128) || page_size <= 0 || page_size % 16 != 0 || num_pages <= 0 || (long long)page_size * num_pages > 0x7fffffffLL) return false;
    auto bytes = [](const void* p) { return static_cast<uint8_t*>(const_cast<void*>(p)); };
    c.k = bytes(k); c.ks = bytes(ks); c.v = bytes(v); c.vs = bytes(vs);
    c.k_scale = k_scale; c.v_scale = v_scale;
    c.kv_heads = kv_heads; c.hd = hd; c.page_size = page_size;
    c.slots = (uint32_t)page_size * (uint32_t)num_pages;
    c.page = FastDiv((uint32_t)page_size);
    return true;
}

}  // namespace

extern "C" {

int fp4_rope_append(const fp4_append_args_t* g) {
    if (!g || !g->qkv_bf16 || !g->cos_tab || !g->sin_tab || !g->positions || !g->slots) return (int)cudaErrorInvalidValue;
    if (!aligned(g->qkv_bf16, 16) || !aligned(g->q_out, 16) || !aligned(g->cos_tab, 4) || !aligned(g->sin_tab, 4) || !aligned(g->positions, 4) || !aligned(g->slots, 4))
        return (int)cudaErrorInvalidValue;
    Append a;
    if (g->tokens < 0 || g->q_heads <= 0 || g->rope_rows <= 0 ||
        !cache_of(a.cache, g->k_codes, g->k_scales, g->v_codes, g->v_scales, g->k_scale, g->v_scale, g->kv_heads, g->head_dim, g->page_size, g->num_pages))
        return (int)cudaErrorInvalidValue;
    const long long heads = (long long)g->q_heads + 2LL * g->kv_heads;
    if (heads > 0x7fffffffLL / 4 || g->tokens > 0x7fffffffLL / (heads * (g->head_dim / 32))) return (int)cudaErrorInvalidValue;
    if (g->tokens == 0) return 0;
    a.qkv = static_cast<const uint16_t*>(g->qkv_bf16);
    a.cos_tab = g->cos_tab; a.sin_tab = g->sin_tab; a.positions = g->positions; a.slots = g->slots;
    a.q_out = static_cast<uint16_t*>(g->q_out);
    a.items = (uint32_t)(g->tokens * heads * (g->head_dim / 32));
    a.q_heads = g->q_heads; a.rope_rows = g->rope_rows;
    a.cph = FastDiv((uint32_t)(g->head_dim / 32));
    a.heads = FastDiv((uint32_t)heads);
    return (int)launch_pdl(fp4_append_kernel, dim3((unsigned)grid_for(a.items)), dim3(THREADS), 0, (cudaStream_t)g->stream, a);
}

int fp4_cache_rows(const fp4_rows_args_t* g) {
    if (!g || !g->slots || !g->k_out || !g->v_out || !aligned(g->slots, 4) || !aligned(g->k_out, 16) || !aligned(g->v_out, 16)) return (int)cudaErrorInvalidValue;
    Rows a;
    if (g->tokens < 0 || !cache_of(a.cache, g->k_codes, g->k_scales, g->v_codes, g->v_scales, g->k_scale, g->v_scale, g->kv_heads, g->head_dim, g->page_size, g->num_pages))
        return (int)cudaErrorInvalidValue;
    if (g->kv_heads > 0x3fffffff / 8 || g->tokens > 0x3fffffffLL / ((long long)g->kv_heads * (g->head_dim / 16))) return (int)cudaErrorInvalidValue;
    if (g->tokens == 0) return 0;
    a.slots = g->slots;
    a.k_out = static_cast<uint16_t*>(g->k_out);
    a.v_out = static_cast<uint16_t*>(g->v_out);
    a.items = (uint32_t)((long long)g->tokens * g->kv_heads * (g->head_dim / 16));
    a.groups = FastDiv((uint32_t)(g->head_dim / 16));
    a.heads = FastDiv((uint32_t)g->kv_heads);
    return (int)launch_pdl(fp4_rows_kernel, dim3((unsigned)grid_for(2 * (size_t)a.items)), dim3(THREADS), 0, (cudaStream_t)g->stream, a);
}

}  // extern "C"
