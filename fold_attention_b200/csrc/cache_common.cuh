// Device helpers of the paged, quantised KV cache: the writers' quantisers and where a row lives.
//
// A row (one token of one head) is handled by D/16 lanes that each own one
// 16-byte unit of every stored plane, so a load is two and a store one 128-bit
// access, and K's XOR swizzle moves whole units. Each fp32 operation the cache
// format specifies is issued as its own round-to-nearest instruction (never
// contracted into an FMA), which makes the planes the bits of the reference's
// torch quantisers (src/fold_attention/decode/cache.py:72-158) whatever the
// batch a row is written with.
#pragma once
#include "common.cuh"

namespace fold {

constexpr int NT = 128;       // threads per CTA
constexpr float INV127 = 0.007874015718698502f;  // fp32(1)/fp32(127)

// Hadamard butterfly over a row split across `LANES` lanes of 16 elements:
// stages 1..8 inside the thread, the rest across lanes, then the 1/sqrt(D)
// scale (reference: utils.py:60-78, decode/quant.py:54-72).
template <int LANES>
__device__ __forceinline__ void rotate16(float (&x)[16], int lane, float hscale) {
#pragma unroll
    for (int h = 1; h < 16; h <<= 1) {
        float y[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if ((i & h) == 0) {
                y[i] = __fadd_rn(x[i], x[i + h]);
                y[i + h] = __fsub_rn(x[i], x[i + h]);
            }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = y[i];
    }
#pragma unroll
    for (int off = 1; off < LANES; off <<= 1) {
        const bool upper = (lane & off) != 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float o = __shfl_xor_sync(0xffffffffu, x[i], off);
            x[i] = upper ? __fsub_rn(o, x[i]) : __fadd_rn(x[i], o);
        }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = __fmul_rn(x[i], hscale);
}

template <int LANES>
__device__ __forceinline__ float row_amax16(const float (&x)[16]) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = fmaxf(m, fabsf(x[i]));
#pragma unroll
    for (int off = 1; off < LANES; off <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    return m;
}

__device__ __forceinline__ uint32_t pack4_s8(int a, int b, int c, int d) {
    return (a & 0xFF) | ((b & 0xFF) << 8) | ((c & 0xFF) << 16) | ((d & 0xFF) << 24);
}

// x = e (a + b/256): plane A from one rounded reciprocal and a multiply,
// plane B from the residual times a rounded 256/e (cache.py:72-78).
__device__ __forceinline__ void int8_planes16(const float (&x)[16], float e, uint4& wa, uint4& wb) {
    const float ie = __fdiv_rn(1.0f, e);
    const float t = __fdiv_rn(256.0f, e);
    int a[16], b[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float u = fmaxf(fminf(__fmul_rn(x[i], ie), 127.0f), -128.0f);
        float pa = rintf(u);
        float r = __fsub_rn(x[i], __fmul_rn(pa, e));
        float w = fmaxf(fminf(__fmul_rn(r, t), 127.0f), -128.0f);
        a[i] = static_cast<int>(pa);
        b[i] = static_cast<int>(rintf(w));
    }
    wa = make_uint4(pack4_s8(a[0], a[1], a[2], a[3]), pack4_s8(a[4], a[5], a[6], a[7]),
                    pack4_s8(a[8], a[9], a[10], a[11]), pack4_s8(a[12], a[13], a[14], a[15]));
    wb = make_uint4(pack4_s8(b[0], b[1], b[2], b[3]), pack4_s8(b[4], b[5], b[6], b[7]),
                    pack4_s8(b[8], b[9], b[10], b[11]), pack4_s8(b[12], b[13], b[14], b[15]));
}

// two fp32 -> packed e4m3x2 (lo in the low byte), round to nearest even, saturating
__device__ __forceinline__ uint32_t cvt_e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ float e4m3_to_float(uint32_t b) {
    // exact: e4m3 -> f16 is a hardware conversion, f16 -> f32 is exact
    uint32_t h2;
    uint16_t s = static_cast<uint16_t>(b & 0xFF);
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(s));
    return __half2float(__ushort_as_half(static_cast<uint16_t>(h2 & 0xFFFF)));
}

// V's two e4m3 planes in units of the layer scale: a = e4m3(clamp(v/e)),
// b = e4m3(clamp((v/e - a) * 8)) (cache.py:81-85).
__device__ __forceinline__ void e4m3_planes16(const float (&v)[16], float ievs, uint4& wa, uint4& wb) {
    uint32_t ca[16], cb[16];
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
        float s0 = __fmul_rn(v[i], ievs), s1 = __fmul_rn(v[i + 1], ievs);
        float c0 = fmaxf(fminf(s0, 448.f), -448.f), c1 = fmaxf(fminf(s1, 448.f), -448.f);
        uint32_t p = cvt_e4m3x2(c0, c1);
        ca[i] = p & 0xFF;
        ca[i + 1] = p >> 8;
        float r0 = __fmul_rn(__fsub_rn(s0, e4m3_to_float(ca[i])), 8.0f);
        float r1 = __fmul_rn(__fsub_rn(s1, e4m3_to_float(ca[i + 1])), 8.0f);
        r0 = fmaxf(fminf(r0, 448.f), -448.f);
        r1 = fmaxf(fminf(r1, 448.f), -448.f);
        uint32_t q = cvt_e4m3x2(r0, r1);
        cb[i] = q & 0xFF;
        cb[i + 1] = q >> 8;
    }
    auto pk = [](const uint32_t* c) { return c[0] | (c[1] << 8) | (c[2] << 16) | (c[3] << 24); };
    wa = make_uint4(pk(ca), pk(ca + 4), pk(ca + 8), pk(ca + 12));
    wb = make_uint4(pk(cb), pk(cb + 4), pk(cb + 8), pk(cb + 12));
}

// A rotated key's planes at pool row `prow`, swizzled by its page slot, and
// its bf16 scale (amax/127 rounded up to bf16, cache.py:97-106).
template <int D>
__device__ __forceinline__ void put_key(const float (&xk)[16], int8_t* ka, int8_t* kb,
                                        __nv_bfloat16* ek, int64_t prow, int off, int lane, bool ok) {
    constexpr int LANES = D / 16;
    constexpr int NU = LANES < 8 ? LANES : 8;
    constexpr int SH = NU == 8 ? 0 : (NU == 4 ? 1 : (NU == 2 ? 2 : 3));
    float e = __fmul_rn(fmaxf(row_amax16<LANES>(xk), 1e-30f), INV127);
    uint32_t hi = (__float_as_uint(e) + 0xFFFFu) >> 16;
    float es = __uint_as_float(hi << 16);
    uint4 wa, wb;
    int8_planes16(xk, es, wa, wb);
    if (ok) {
        int64_t addr = prow * D + ((lane ^ ((off >> SH) & (NU - 1))) * 16);
        *reinterpret_cast<uint4*>(ka + addr) = wa;
        *reinterpret_cast<uint4*>(kb + addr) = wb;
        if (lane == 0) reinterpret_cast<uint16_t*>(ek)[prow] = static_cast<uint16_t>(hi);
    }
}

template <int D, bool V8, bool F16>
__device__ __forceinline__ void put_value(const float (&xv)[16], const uint4 (&wv)[2], void* va,
                                          void* vb, int64_t prow, int lane, bool ok, float ievs) {
    if constexpr (V8) {
        uint4 wa, wb;
        e4m3_planes16(xv, ievs, wa, wb);
        if (ok) {
            int64_t addr = prow * D + lane * 16;
            *reinterpret_cast<uint4*>(static_cast<uint8_t*>(va) + addr) = wa;
            *reinterpret_cast<uint4*>(static_cast<uint8_t*>(vb) + addr) = wb;
        }
    } else {
        if (ok) {
            uint4* dst = reinterpret_cast<uint4*>(static_cast<uint8_t*>(va) + (prow * D + lane * 16) * 2);
            if constexpr (F16) {
                // the pool is bf16: an fp16 token is rounded to it once
                dst[0] = make_uint4(pack_bf16x2(xv[0], xv[1]), pack_bf16x2(xv[2], xv[3]),
                                    pack_bf16x2(xv[4], xv[5]), pack_bf16x2(xv[6], xv[7]));
                dst[1] = make_uint4(pack_bf16x2(xv[8], xv[9]), pack_bf16x2(xv[10], xv[11]),
                                    pack_bf16x2(xv[12], xv[13]), pack_bf16x2(xv[14], xv[15]));
            } else {
                dst[0] = wv[0];
                dst[1] = wv[1];
            }
        }
    }
}

}  // namespace fold
