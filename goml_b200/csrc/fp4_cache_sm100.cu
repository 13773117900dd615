// fp4_cache_sm100.cu — rows into and out of a KV cache held in 4 bits (fp4_rope_append and fp4_cache_rows, include/fp8_block.h).
//
// Both are one pass over their rows, a thread to 16 dims of one (token, head).  HBM-bound: an append reads 2 bytes a value of the projection and writes 2 of the queries and
// 0.56 of keys and values; what keeps it from the memory's rate is the rounding of keys and values (about 290 instructions of a warp for 32 x 16 of them, 350 where ties are to be expected)
// and then warps with loads in flight, so a thread takes few values and few registers.  (32 dims to a thread without the exchange between two: 24 tokens 3.3 us for 2.0, 4000 of 32
// query heads on 8 21.2 for 20.3, 16384 of 32 on 32 146 for 158.)
//
// Measured: 16384 tokens, 32 query heads on 8 of 128, appended in 73 us = 5.0 TB/s and read back in 18.6 (4.6 TB/s); 32 on 32 160 us (3.9; 175 before the question whether anything is near a border) and 62 (5.6).
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/fp8_block.h"
#include "pdl.cuh"
#include "row_items.cuh"

namespace {

using namespace sm100;

constexpr int THREADS = 256;
constexpr int CTAS_PER_SM = 4;   // as many as are resident: with two and more rounds of them 16384 tokens take 3 to 15 us longer

int grid_for(size_t items) {
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    const size_t blocks = (items + THREADS - 1) / THREADS, cap = (size_t)sms * CTAS_PER_SM;
    return (int)(blocks < cap ? blocks : cap);
}
bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// Rounding a quotient may hide on which side of a border between two codes it lies.  Borders are numbers whose last DROP bits of 23 are zero; where q lies within a few units in the
// last place of such a number m, what it is replaced by is m moved by the residual of m times 2^10 of its size: the residual's sign is exact, its size is below 2^-20 of the
// quotient there, and a quotient that is m stays m.
// (Not a branch: values of few bits are near borders in a warp as often as not.)
template <int DROP>
__device__ __forceinline__ float border_near(float q, bool& near) {
    const uint32_t bits = __float_as_uint(q), at = (bits + (1u << (DROP - 1))) & ~((1u << DROP) - 1u);
    near = bits - at + 8u <= 16u;
    return __uint_as_float(at);
}

// two at a time
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 neg(float2 a) { return make_float2(-a.x, -a.y); }

// to an ulp, which is less than what counts as near a border
__device__ __forceinline__ float reciprocal(float x) {
    float r;
    asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// Values of a tensor whose scale is below FEW, and their divisors, are taken RAISE times: reciprocals and residuals then stay in fp32's normal range, and 2^10 times a reciprocal below
// infinity.  (Raising is exact, but for what becomes an infinity: that is beyond every border.  The least block scale is 2^-9.)
constexpr float FEW = 0x1p-91f, RAISE = 0x1p64f;
// A tensor scale and what the quotients by it need
struct TensorScale {
    float s, raise, six, six_rest, inv_six;   // six + six_rest is 6 s exactly, raised
    __device__ __forceinline__ TensorScale(float scale, float raise_) : s(scale), raise(raise_) {
        const float r = scale * raise;
        six = __fmul_rn(6.f, r);
        six_rest = __fmaf_rn(6.f, r, -six);
        inv_six = reciprocal(six);
    }
};

// e4m3(a / 6s), a >= 0.  Borders between e4m3 numbers have at most five significant bits.
__device__ __forceinline__ uint32_t block_scale(float a, const TensorScale& ts) {
    bool near;
    float q = __fmul_rn(a, ts.inv_six);
    const float m = border_near<19>(q, near);
    const float rest = __fmaf_rn(-m, ts.six_rest, __fmaf_rn(-m, ts.six, a));   // the first is exact: a and m * six cancel to their last bits
    if (near && q < 1024.f) q = __fmaf_rn(rest * 1024.f, ts.inv_six, m);   // (an infinity saturates)
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(q));
    return r & 0xffu;
}
__device__ __forceinline__ float e4m3_to_f32(uint32_t b) {
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(r) : "r"(b));
    return __half2float(__low2half(*reinterpret_cast<const __half2*>(&r)));
}
__device__ __forceinline__ float max_abs(float m, float y) {   // a NaN stays
    float r;
    asm("{\n\t.reg .f32 a;\n\tabs.f32 a, %2;\n\tmax.NaN.f32 %0, %1, a;\n\t}" : "=f"(r) : "f"(m), "f"(y));
    return r;
}
// Eight values of a group in codes.  Borders between codes have at most three significant bits.
struct GroupScale {
    float d, inv;
    bool none;
    __device__ __forceinline__ GroupScale(uint32_t b, const TensorScale& ts) {
        d = __fmul_rn(e4m3_to_f32(b), ts.s);
        none = !(d >= 1.1754943508222875e-38f);   // zeros; of a NaN, too
        d *= ts.raise;
        inv = reciprocal(d);
    }
};
__device__ __forceinline__ uint32_t codes8(const float* q) {
    uint32_t w;
    asm("{\n\t.reg .b8 a, b, c, d;\n\tcvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\tmov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(w)
        : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]), "f"(q[4]), "f"(q[5]), "f"(q[6]), "f"(q[7]));
    return w;
}
// ties: whether values halfway between two codes are to be expected
__device__ __forceinline__ uint32_t quantise8(float* y, const GroupScale& g, bool largest, bool ties) {
    if (!ties) {   // a value near a border is one in 100000: whether there is any costs half of what is done about it
        float q[8];
        uint32_t nearest = 0xffffffffu;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const float2 a = mul2(make_float2(y[i], y[i + 1]), make_float2(g.inv, g.inv));
            q[i] = a.x;
            q[i + 1] = a.y;
            nearest = min(nearest, min((__float_as_uint(a.x) + 8u) & 0x1fffffu, (__float_as_uint(a.y) + 8u) & 0x1fffffu));
        }
        if (nearest > 16u) return g.none ? 0u : codes8(q);
    }
    if (__builtin_expect(largest, 0)) {   // the largest block scale: what is beyond it saturates, infinities among it
#pragma unroll
        for (int i = 0; i < 8; i++) y[i] = fminf(fmaxf(y[i], -8.f * g.d), 8.f * g.d);
    }
    const float inv_1024 = g.inv * 1024.f;
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const float2 x = make_float2(y[i], y[i + 1]);
        bool near0, near1;
        const float2 a = mul2(x, make_float2(g.inv, g.inv));
        const float2 m = make_float2(border_near<21>(a.x, near0), border_near<21>(a.y, near1));
        const float2 moved = fma2(fma2(neg(m), make_float2(g.d, g.d), x), make_float2(inv_1024, inv_1024), m);
        q[i] = copysignf(near0 ? moved.x : a.x, x.x);   // of a zero, too
        q[i + 1] = copysignf(near1 ? moved.y : a.y, x.y);
    }
    return g.none ? 0u : codes8(q);
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
    uint32_t items;   // tokens * heads of a row * hd / 16
    int q_heads, rope_rows;
    bool one_round;
    FastDiv pieces, heads;   // 16-dim pieces of a head, heads of a row
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
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}

// RoPE pairs dim i with dim i + hd/2: of queries and keys a thread takes 8 dims of one half and their partners of the other, and two threads side by side have two groups
// of 16, whose scales they find one each; of values it takes a group.
__global__ void __launch_bounds__(THREADS, CTAS_PER_SM) fp4_append_kernel(const Append a) {
    pdl_wait();
    pdl_trigger();
    const int hd = a.cache.hd, half = hd / 2, kv = a.cache.kv_heads, odd = threadIdx.x & 1;
    const float k_scale = ld_f32(a.cache.k_scale), v_scale = ld_f32(a.cache.v_scale);
    // a warp's threads stay together: items come in pairs of threads, and a row has a whole number of those
    for (uint32_t it0 = blockIdx.x * THREADS + (threadIdx.x & ~31u); it0 < a.items; it0 += gridDim.x * THREADS) {
        const bool there = it0 + (threadIdx.x & 31) < a.items;
        const uint32_t it = there ? it0 + (threadIdx.x & 31) : it0;
        uint32_t r, c, token, head;
        a.pieces.divmod(it, r, c);
        a.heads.divmod(r, token, head);
        const bool is_q = (int)head < a.q_heads, is_v = (int)head >= a.q_heads + kv;
        const int d0 = is_v ? 16 * c : 8 * c, apart = is_v ? 8 : half;
        const uint16_t* x = a.qkv + (size_t)r * hd + d0;
        const uint4 x0 = ld128(x), x1 = ld128(x + apart);
        const int pos = ld_s32(a.positions + token), slot = ld_s32(a.slots + token);
        const bool active = pos >= 0 && pos < a.rope_rows;
        float y[16];
        bf16x8_to_f32(x0, y);
        bf16x8_to_f32(x1, y + 8);
        if (!is_v && active) {
            const float* cs = a.cos_tab + (size_t)pos * half + 8 * c;
            const float* sn = a.sin_tab + (size_t)pos * half + 8 * c;
#pragma unroll
            for (int j = 0; j < 8; j += 4) {
                const float4 c4 = ld128f(cs + j), s4 = ld128f(sn + j);
                const float cc[4] = {c4.x, c4.y, c4.z, c4.w}, ss[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
                for (int i = j; i < j + 4; i++) {   // (packed products and sums are contracted into fused ones, whatever their rounding says)
                    const float y0 = y[i], y1 = y[8 + i];
                    y[i] = __fsub_rn(__fmul_rn(y0, cc[i - j]), __fmul_rn(y1, ss[i - j]));
                    y[8 + i] = __fadd_rn(__fmul_rn(y0, ss[i - j]), __fmul_rn(y1, cc[i - j]));
                }
            }
        }
        if (is_q && there && a.q_out) {
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; i++) w[i] = active ? bf16x2(y[2 * i], y[2 * i + 1]) : 0u;
            uint16_t* q = a.q_out + ((size_t)token * a.q_heads + head) * hd + d0;
            *reinterpret_cast<uint4*>(q) = make_uint4(w[0], w[1], w[2], w[3]);
            *reinterpret_cast<uint4*>(q + apart) = make_uint4(w[4], w[5], w[6], w[7]);
        }
        const bool stores = !is_q && there && active && slot >= 0 && (uint32_t)slot < a.cache.slots;
        if (!__any_sync(0xffffffffu, stores)) continue;
        const float scale = is_v ? v_scale : k_scale;
        float raise = 1.f;
        if (__builtin_expect(scale < FEW, 0)) {
            raise = RAISE;
#pragma unroll
            for (int i = 0; i < 16; i++) y[i] *= RAISE;
        }
        float top[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 8; i++) {
            top[0] = max_abs(top[0], y[i]);
            top[1] = max_abs(top[1], y[8 + i]);
        }
        const float other[2] = {__shfl_xor_sync(0xffffffffu, top[0], 1), __shfl_xor_sync(0xffffffffu, top[1], 1)};
        const TensorScale ts(scale, raise);
        // of keys the first thread has the scale of the first half's group, the second that of the other's; of values each its own
        const float mine_top = is_v ? max_abs(top[0], top[1]) : odd ? max_abs(top[1], other[1]) : max_abs(top[0], other[0]);
        const uint32_t mine = isnan(mine_top) ? 0x7fu : block_scale(mine_top, ts), theirs = __shfl_xor_sync(0xffffffffu, mine, 1);
        if (!stores) continue;
        const GroupScale g0(is_v || !odd ? mine : theirs, ts), g1(is_v || odd ? mine : theirs, ts);
        const size_t row = a.cache.row(slot, (int)head - a.q_heads - (is_v ? kv : 0));
        // bf16 by a scale of few bits; what RoPE has turned has all of its bits.  (And where a step is one round of threads, which the question only makes longer: 24 tokens 2.12 us for 2.17.)
        const bool ties = a.one_round || (is_v && (__float_as_uint(ts.s) & 0x7ffffu) == 0);
        uint8_t* const codes = (is_v ? a.cache.v : a.cache.k) + row * half + d0 / 2;
        *reinterpret_cast<uint32_t*>(codes) = quantise8(y, g0, (is_v || !odd ? mine : theirs) == 0x7eu, ties);
        *reinterpret_cast<uint32_t*>(codes + apart / 2) = quantise8(y + 8, g1, (is_v || odd ? mine : theirs) == 0x7eu, ties);
        if (is_v) *a.cache.v_scale_at(row, c) = (uint8_t)mine;
        else *a.cache.k_scale_at(row, (odd ? half / 16 : 0) + c / 2) = (uint8_t)mine;
    }
}

struct Rows {
    const int32_t* slots;
    uint16_t *k_out, *v_out;
    Cache cache;
    uint32_t items;   // tokens * kv heads * hd / 16, of keys and then as many of values
    FastDiv groups, heads;
};
// Four items to a thread side by side: one is 9 bytes, too few to keep the memory busy (16384 tokens, 32 heads of 128: one 79 us)
constexpr int ROWS_SIDE = 4;
__global__ void __launch_bounds__(THREADS) fp4_rows_kernel(const Rows a) {
    pdl_wait();
    pdl_trigger();
    const int hd = a.cache.hd;
    const float k_scale = ld_f32(a.cache.k_scale), v_scale = ld_f32(a.cache.v_scale);
    const uint32_t step = gridDim.x * THREADS;
    for (uint32_t i0 = blockIdx.x * THREADS + threadIdx.x; i0 < 2 * a.items; i0 += ROWS_SIDE * step) {
        int slot[ROWS_SIDE];
        uint32_t head[ROWS_SIDE], group[ROWS_SIDE], w[ROWS_SIDE][2], bytes[ROWS_SIDE];
#pragma unroll
        for (int k = 0; k < ROWS_SIDE; k++) {
            const uint32_t i = i0 + k * step, it = i >= a.items ? i - a.items : i;
            uint32_t r, token;
            a.groups.divmod(it, r, group[k]);
            a.heads.divmod(r, token, head[k]);
            slot[k] = i < 2 * a.items ? ld_s32(a.slots + token) : -1;
        }
#pragma unroll
        for (int k = 0; k < ROWS_SIDE; k++) {
            w[k][0] = w[k][1] = bytes[k] = 0u;
            if (slot[k] < 0 || (uint32_t)slot[k] >= a.cache.slots) continue;
            const bool is_v = i0 + k * step >= a.items;
            const size_t row = a.cache.row(slot[k], (int)head[k]);
            const uint8_t* codes = (is_v ? a.cache.v : a.cache.k) + row * (hd / 2) + 8 * group[k];
            asm volatile("ld.global.v2.u32 {%0,%1}, [%2];" : "=r"(w[k][0]), "=r"(w[k][1]) : "l"(codes) : "memory");
            uint16_t b;
            asm volatile("ld.global.u8 %0, [%1];" : "=h"(b) : "l"(is_v ? a.cache.v_scale_at(row, group[k]) : a.cache.k_scale_at(row, group[k])) : "memory");
            bytes[k] = b;
        }
#pragma unroll
        for (int k = 0; k < ROWS_SIDE; k++) {
            const uint32_t i = i0 + k * step;
            if (i >= 2 * a.items) break;
            const bool is_v = i >= a.items;
            const float s = is_v ? v_scale : k_scale, bs = e4m3_to_f32(bytes[k]);
            float y[16];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                uint32_t x[4];
                asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
                    "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
                    : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                    : "r"(w[k][h]));
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x[j]));
                    y[8 * h + 2 * j] = __fmul_rn(__fmul_rn(f.x, bs), s);   // the first product is exact
                    y[8 * h + 2 * j + 1] = __fmul_rn(__fmul_rn(f.y, bs), s);
                }
            }
            if (slot[k] < 0 || (uint32_t)slot[k] >= a.cache.slots) {   // whatever the tensor scale is
#pragma unroll
                for (int j = 0; j < 16; j++) y[j] = 0.f;
            }
            store_bf16x16((is_v ? a.v_out : a.k_out) + (size_t)(is_v ? i - a.items : i) * 16, y);
        }
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
    if (!aligned(g->qkv_bf16, 16) || !aligned(g->q_out, 16) || !aligned(g->cos_tab, 16) || !aligned(g->sin_tab, 16) || !aligned(g->positions, 4) || !aligned(g->slots, 4))
        return (int)cudaErrorInvalidValue;
    Append a;
    if (g->tokens < 0 || g->q_heads <= 0 || g->rope_rows <= 0 ||
        !cache_of(a.cache, g->k_codes, g->k_scales, g->v_codes, g->v_scales, g->k_scale, g->v_scale, g->kv_heads, g->head_dim, g->page_size, g->num_pages))
        return (int)cudaErrorInvalidValue;
    const long long heads = (long long)g->q_heads + 2LL * g->kv_heads;
    if (heads > 0x7fffffffLL / 8 || g->tokens > (0x7fffffffLL - 32) / (heads * (g->head_dim / 16))) return (int)cudaErrorInvalidValue;
    if (g->tokens == 0) return 0;
    a.qkv = static_cast<const uint16_t*>(g->qkv_bf16);
    a.cos_tab = g->cos_tab; a.sin_tab = g->sin_tab; a.positions = g->positions; a.slots = g->slots;
    a.q_out = static_cast<uint16_t*>(g->q_out);
    a.items = (uint32_t)(g->tokens * heads * (g->head_dim / 16));
    a.q_heads = g->q_heads; a.rope_rows = g->rope_rows;
    a.pieces = FastDiv((uint32_t)(g->head_dim / 16));
    a.heads = FastDiv((uint32_t)heads);
    const int grid = grid_for(a.items);
    a.one_round = (size_t)grid * THREADS >= a.items;
    return (int)launch_pdl(fp4_append_kernel, dim3((unsigned)grid), dim3(THREADS), 0, (cudaStream_t)g->stream, a);
}

int fp4_cache_rows(const fp4_rows_args_t* g) {
    if (!g || !g->slots || !g->k_out || !g->v_out || !aligned(g->slots, 4) || !aligned(g->k_out, 32) || !aligned(g->v_out, 32)) return (int)cudaErrorInvalidValue;
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
    // few items: one to a thread (24 tokens, 8 heads of 128: 1.9 us, four to a thread 2.6)
    const size_t items = 2 * (size_t)a.items;
    const int few = grid_for(items);
    return (int)launch_pdl(fp4_rows_kernel, dim3((unsigned)((size_t)few * THREADS >= items ? few : grid_for((items + ROWS_SIDE - 1) / ROWS_SIDE))), dim3(THREADS), 0, (cudaStream_t)g->stream, a);
}

}  // extern "C"
