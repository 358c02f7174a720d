// tqb_quant_row.cuh — one token-head of the cache store: value quantisation and
// the slot writes, shared by the store and the append kernels.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "tqb_common.cuh"
#include "tqb_internal.h"

namespace tqb {

// a / b rounded to nearest even, from y = RN(1/b): Markstein's FMA
// iteration (P. Markstein, "Computation of elementary functions on the IBM
// RISC System/6000 processor", IBM J. Res. Dev. 34(1), 1990).  q0 = RN(a y)
// is within 1.5 ulp of a/b; the first correction makes it faithful, after
// which the residual a - b q1 is exact and the second correction rounds
// correctly.  Holds for b and 1/b normal and a quotient far from the
// subnormal range; below that the store maps every candidate to code 0.
__device__ __forceinline__ float div_rn_by_rcp(float a, float b, float y) {
    const float q0 = __fmul_rn(a, y);
    const float r0 = __fmaf_rn(-b, q0, a);
    const float q1 = __fmaf_rn(r0, y, q0);
    const float r1 = __fmaf_rn(-b, q1, a);
    return __fmaf_rn(r1, y, q1);
}

// Byte stores of a little-endian value (3-bit streams, 2-byte-aligned slots).
__device__ __forceinline__ void st_bytes3(uint8_t* p, uint32_t v) {
    p[0] = (uint8_t)v;
    p[1] = (uint8_t)(v >> 8);
    p[2] = (uint8_t)(v >> 16);
}
__device__ __forceinline__ void st_u16x2(uint8_t* p, uint32_t v) {
    reinterpret_cast<unsigned short*>(p)[0] = (unsigned short)v;
    reinterpret_cast<unsigned short*>(p)[1] = (unsigned short)(v >> 16);
}

// The value codes of one token-head: 16 lanes (half a warp), 8 consecutive dims
// each.  All 32 lanes call it.  bits: this lane's 8 codes; scale and vmin are
// the row's, on every lane.
struct ValueRow {
    uint32_t bits;
    float scale, vmin;
};
template <bool V3>
__device__ __forceinline__ ValueRow quantise_values(const float (&vs)[8]) {
    constexpr unsigned kFull = 0xffffffffu;
    float vmin = vs[0], vmax = vs[0];
#pragma unroll
    for (int j = 1; j < 8; j++) {
        vmin = fminf(vmin, vs[j]);
        vmax = fmaxf(vmax, vs[j]);
    }
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
        vmin = fminf(vmin, __shfl_xor_sync(kFull, vmin, o));
        vmax = fmaxf(vmax, __shfl_xor_sync(kFull, vmax, o));
    }
    // 3-bit values (reference/soa_store.py:49-84): 7 levels, codes packed
    // little-endian at bit 3d; 4-bit: 15 levels, two codes per byte.
    // scale = max((max - min) / levels, 1e-8): a range below 1e-7 ends at the
    // floor, so the division only matters for normal ranges, where the FMA
    // iteration on RN(1/levels) is exact; an infinite range stays infinite.
    constexpr int vtop = V3 ? 7 : 15;
    constexpr float kRcpTop = 1.0f / (float)vtop;  // correctly rounded at compile time
    const float range = __fsub_rn(vmax, vmin);
    float scale = range < INFINITY ? div_rn_by_rcp(range, (float)vtop, kRcpTop) : range;
    scale = scale > 1e-8f ? scale : 1e-8f;
    float qv[8];
    if (isfinite(scale)) {  // uniform over the half-warp
        const float y = __frcp_rn(scale);
#pragma unroll
        for (int j = 0; j < 8; j++) qv[j] = div_rn_by_rcp(__fsub_rn(vs[j], vmin), scale, y);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) qv[j] = __fdiv_rn(__fsub_rn(vs[j], vmin), scale);
    }
    uint32_t vbits = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        int q = __float2int_rz(__fadd_rn(qv[j], 0.5f));
        q = q < 0 ? 0 : (q > vtop ? vtop : q);
        vbits |= (uint32_t)q << ((V3 ? 3 : 4) * j);
    }
    return ValueRow{vbits, scale, vmin};
}

// The slot of token-head (off, h) in the block at `base`: value codes, fp16
// key norm, value scale and zero.
template <int L>
struct SlotAt {
    uint8_t *key, *value, *norm, *scale, *zero;
    __device__ __forceinline__ SlotAt(uint8_t* base, uint32_t off, uint32_t h, int H, int64_t pos_stride,
                                      int64_t head_stride) {
        if constexpr (layout_is_aos(L)) {
            // [key codes | fp16 norm | value codes | fp16 scale | fp16 zero]
            // (reference/aos_store.py:26-116, :183-203, :296-325)
            key = base + (size_t)off * pos_stride + (size_t)h * head_stride;
            value = key + aos_val_off(L);
            norm = key + aos_norm_off(L);
            scale = key + aos_scale_off(L);
            zero = scale + 2;
        } else {
            constexpr int kKey = aos_key_bytes(L), kRow = kKey + val_code_bytes(L), kFields = layout_fp8_keys(L) ? 2 : 3;
            key = base + (size_t)off * ((size_t)H * kRow) + (size_t)h * kRow;
            value = key + kKey;
            norm = base + (size_t)kBlockSize * H * kRow + ((size_t)h * kFields * kBlockSize + off) * 2;
            scale = norm + (kFields - 2) * kBlockSize * 2;
            zero = scale + kBlockSize * 2;
        }
    }
};

// Half a warp's value codes (lane m of 16: dims 8m .. 8m + 7) and their grid.
template <int L>
__device__ __forceinline__ void write_values(const SlotAt<L>& at, int m, const ValueRow& v) {
    if constexpr (layout_3bit_values(L))
        st_bytes3(at.value + 3 * m, v.bits);
    else if constexpr (L == TQB_LAYOUT_SOA_K8)
        reinterpret_cast<uint32_t*>(at.value)[m] = v.bits;  // 4-byte aligned rows (checked on the host)
    else
        st_u16x2(at.value + 4 * m, v.bits);
    if (m == 0) {
        *reinterpret_cast<unsigned short*>(at.scale) = __half_as_ushort(__float2half_rn(v.scale));
        *reinterpret_cast<unsigned short*>(at.zero) = __half_as_ushort(__float2half_rn(v.vmin));
    }
}

// Writes one token-head of layout L into token `off` of the block at `base`:
// lane m of 16 holds dims 8m .. 8m + 7, their key codes in kbits (e4m3 keys:
// the bytes in klo, khi) and value codes in v; vn_h is the fp16 key norm as
// stored (SoA: with the norm correction folded in, AoS: the raw norm,
// reference/aos_store.py:317-325).  H KV heads, this one is h.
template <int L>
__device__ __forceinline__ void write_row(uint8_t* base, uint32_t off, uint32_t h, int H, int64_t pos_stride,
                                          int64_t head_stride, int m, uint32_t kbits, uint32_t klo, uint32_t khi,
                                          const ValueRow& v, unsigned short vn_h) {
    const SlotAt<L> at(base, off, h, H, pos_stride, head_stride);
    if constexpr (L == TQB_LAYOUT_SOA_K8) {
        reinterpret_cast<uint32_t*>(at.key)[2 * m] = klo;
        reinterpret_cast<uint32_t*>(at.key)[2 * m + 1] = khi;
    } else if constexpr (layout_fp8_keys(L)) {
        st_u16x2(at.key + 8 * m, klo);
        st_u16x2(at.key + 8 * m + 4, khi);
    } else if constexpr (layout_3bit_keys(L)) {
        st_bytes3(at.key + 3 * m, kbits);  // dims 8m .. 8m+7 = bits 24m .. 24m+23 of the stream
    } else {
        st_u16x2(at.key + 4 * m, kbits);
    }
    if (!layout_fp8_keys(L) && m == 0) *reinterpret_cast<unsigned short*>(at.norm) = vn_h;
    write_values<L>(at, m, v);
}

}  // namespace tqb
