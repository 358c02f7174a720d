// tqb_rot_mma.cuh — 16 rows times 32 columns of the rotation by one warp, on the
// register-operand tensor cores, for kernels that must start without staging R.
//
// Every operand is split into bf16 parts of 8 bits, which keep fp32's range: R
// into three, the rows into as many as their numbers need; the products down to
// 2^-16 of the first are summed in fp32 (dropped terms: 2^-24 of the row and
// column lengths).  A product's 16 summands may come in any order, and its
// columns too, so lane (g, c) takes the four consecutive dims k + 4c .. + 3 and
// the columns n0 + 4g .. + 3 (one per tile): R, rows and results move in 16-byte
// accesses, a quarter of the loads of the fragments' own order (a window of
// 1024 tokens, 64 x 32 heads, rotation included: 45.9 us in that order, 44.5 so;
// the append of 128 tokens 15.7 and 15.2).
#pragma once
#include <cuda_bf16.h>

#include <cstdint>

#include "tqb_common.cuh"

namespace tqb {

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The next bf16 part of a pair of numbers, which keep the rest.
__device__ __forceinline__ uint32_t take_bf16(float& x, float& y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    x -= __low2float(h);
    y -= __high2float(h);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Sums of a warp's 16 x 32 outputs: of the products of the first parts, and of
// the others (2^-8 of them).
struct RotSums {
    float first[4][4] = {}, small[4][4] = {};
    // Output (row g + 8 i, columns n0 + 8c + 4j .. + 3).
    __device__ __forceinline__ float4 get(int i, int j) const {
        const int e = 2 * i + j;
        return make_float4(first[0][e] + small[0][e], first[1][e] + small[1][e], first[2][e] + small[2][e],
                           first[3][e] + small[3][e]);
    }
};

// Asks for the warp's 32 columns of R, while the rows are on their way (the
// append of one token: 10.1 us without, 9.6 with; of 128: 15.2 and 15.7).
__device__ __forceinline__ void rot_prefetch(const float* R, int n0, int lane) {
#pragma unroll
    for (int i = 0; i < kHeadDim; i += 32)
        asm volatile("prefetch.global.L1 [%0];\n" ::"l"(R + (i + lane) * kHeadDim + n0));
}

// Dims k .. k + 15 of the sum.  x: dims k + 4c .. + 3 of rows g and g + 8, in
// kParts bf16 parts; R: the rotation at (row 4c, column n0 + 4g).  kOutside:
// the full-size products are added up outside the tensor core, which truncates
// the sum it adds to.
template <int kParts, bool kOutside>
__device__ __forceinline__ void rot_step(RotSums& s, const float* R, int k, float4 x0, float4 x1) {
    float4 b[4];
#pragma unroll
    for (int i = 0; i < 4; i++) b[i] = __ldg(reinterpret_cast<const float4*>(R + (k + i) * kHeadDim));
    uint32_t a[kParts][4];
#pragma unroll
    for (int p = 0; p < kParts; p++) {
        a[p][0] = take_bf16(x0.x, x0.y);
        a[p][1] = take_bf16(x1.x, x1.y);
        a[p][2] = take_bf16(x0.z, x0.w);
        a[p][3] = take_bf16(x1.z, x1.w);
    }
#pragma unroll
    for (int q = 0; q < 3; q++)
#pragma unroll
        for (int n = 0; n < 4; n++) {
            float &u0 = (&b[0].x)[n], &u1 = (&b[1].x)[n], &u2 = (&b[2].x)[n], &u3 = (&b[3].x)[n];
            const uint32_t b0 = take_bf16(u0, u1), b1 = take_bf16(u2, u3);
#pragma unroll
            for (int p = 0; p < kParts; p++) {
                if (p + q == 0 && kOutside) {
                    float d[4] = {};
                    mma_bf16(d, a[0], b0, b1);
#pragma unroll
                    for (int i = 0; i < 4; i++) s.first[n][i] += d[i];
                } else if (p + q < 3 || kParts == 2) {
                    mma_bf16(p + q == 0 ? s.first[n] : s.small[n], a[p], b0, b1);
                }
            }
        }
}

}  // namespace tqb
