// Arithmetic shared by the attention kernels: operand types, exponentials on two pipes, packed f32 instructions.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace h3b {

// The two 16-bit operand types: bf16 (the benchmark's residual-stream type) and f16 (what the reference's
// own f16 attention entry points stage in: three more mantissa bits in Q, K, V and in the probabilities).
template <typename T> struct Elem;
template <> struct Elem<__nv_bfloat16> {
    static constexpr uint32_t FMT = 1;   // tcgen05 kind::f16 operand format code
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<uint32_t *>(&h);
    }
};
template <> struct Elem<__half> {
    static constexpr uint32_t FMT = 0;
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<uint32_t *>(&h);
    }
};

__device__ __forceinline__ float ex2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 2^x for two values on the FMA pipe instead of the special-function unit (which is the unit the softmax
// saturates: 16 results per clock and SM against 128 FMA lanes).  x is clamped to >= -127, split into
// floor and fraction by adding 1.5 * 2^23 with round-down (the floor lands in the low mantissa bits), the
// fraction goes through a degree-3 minimax polynomial (relative error 8.6e-5, far below the rounding of the
// probabilities to 16 bits) and the floor is added to the exponent field.  Packed two-wide f32 instructions.
__device__ __forceinline__ void ex2_emu2(float &p0, float &p1, float x0, float x1) {
    x0 = fmaxf(x0, -127.0f);
    x1 = fmaxf(x1, -127.0f);
    uint32_t r0, r1, q0, q1;
    asm("{\n\t.reg .b64 x, m, r, b, f, p, c;\n\t"
        "mov.b64 x, {%4, %5};\n\t"
        "mov.b64 m, {%6, %6};\n\t"
        "add.rm.ftz.f32x2 r, x, m;\n\t"
        "sub.rn.ftz.f32x2 b, r, m;\n\t"
        "sub.rn.ftz.f32x2 f, x, b;\n\t"
        "mov.b64 p, {%7, %7};\n\t"
        "mov.b64 c, {%8, %8};\n\t"
        "fma.rn.ftz.f32x2 p, p, f, c;\n\t"
        "mov.b64 c, {%9, %9};\n\t"
        "fma.rn.ftz.f32x2 p, p, f, c;\n\t"
        "mov.b64 c, {%10, %10};\n\t"
        "fma.rn.ftz.f32x2 p, p, f, c;\n\t"
        "mov.b64 {%0, %1}, r;\n\t"
        "mov.b64 {%2, %3}, p;\n\t}"
        : "=r"(r0), "=r"(r1), "=r"(q0), "=r"(q1)
        : "f"(x0), "f"(x1), "f"(12582912.0f), "f"(0.07706703990697861f), "f"(0.22764499485492706f),
          "f"(0.6951167583465576f), "f"(1.0f));
    p0 = __uint_as_float(q0 + (r0 << 23));
    p1 = __uint_as_float(q1 + (r1 << 23));
}

// max of three (one instruction on sm_100)
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// two-wide f32 FMA / add: one issue slot for two independent IEEE operations
__device__ __forceinline__ void fma2(float &d0, float &d1, float a0, float a1, float b, float c) {
    asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\t"
        "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %4};\n\tmov.b64 rc, {%5, %5};\n\t"
        "fma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d0), "=f"(d1)
        : "f"(a0), "f"(a1), "f"(b), "f"(c));
}
__device__ __forceinline__ void add2(float &d0, float &d1, float a0, float a1) {
    asm("{\n\t.reg .b64 ra, rd;\n\t"
        "mov.b64 rd, {%0, %1};\n\tmov.b64 ra, {%2, %3};\n\t"
        "add.rn.f32x2 rd, rd, ra;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "+f"(d0), "+f"(d1)
        : "f"(a0), "f"(a1));
}

}  // namespace h3b
