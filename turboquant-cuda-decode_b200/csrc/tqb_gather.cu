// tqb_gather.cu — cached keys and values of chosen slots, dequantised.
//
//     key[n, h, :]   = c[code] * norm     (Lloyd-Max keys; AoS: c / |c| * norm)
//                      or the e4m3 numbers themselves,
//     value[n, h, :] = code * scale + zero,
// rounded once to the output type; rows of a negative or out-of-range slot
// are zeros.  The reference's counterpart dequantises a whole sequence for a
// later chunk of its prefill (reference/soa_decode_v1.py:322-454).  The keys
// stay in the rotated basis: the chunk's queries are rotated instead, one row
// per head and token rather than one per cached token.
//
// One pass: 134 bytes (or 196, 118, 102) read and 512 written per token-head
// with 16-bit outputs, so HBM writes bound it.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "tqb_common.cuh"
#include "tqb_internal.h"

namespace tqb {

namespace {

constexpr int kGatherWarps = 8;

__device__ __forceinline__ uint32_t ldu16(const uint8_t* p) {
    return __ldg(reinterpret_cast<const unsigned short*>(p));
}
__device__ __forceinline__ uint32_t ld_bytes3(const uint8_t* p) {
    return (uint32_t)__ldg(p) | ((uint32_t)__ldg(p + 1) << 8) | ((uint32_t)__ldg(p + 2) << 16);
}

// Eight consecutive numbers in the output type (16-byte or 32-byte aligned
// for the vector form).
template <typename T, bool VEC>
__device__ __forceinline__ void put8(T* p, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        if constexpr (VEC) {
            reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            for (int j = 0; j < 8; j++) p[j] = v[j];
        }
    } else {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if constexpr (sizeof(T) == 2 && __is_same(T, __half)) {
                w[j] = h2_as_u32(__floats2half2_rn(v[2 * j], v[2 * j + 1]));
            } else {
                const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
                w[j] = *reinterpret_cast<const uint32_t*>(&b);
            }
        }
        if constexpr (VEC) {
            *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            unsigned short* q = reinterpret_cast<unsigned short*>(p);
            for (int j = 0; j < 8; j++) q[j] = (unsigned short)(w[j >> 1] >> (16 * (j & 1)));
        }
    }
}

// Half a warp per token-head, lane m of 16 on dims 8m .. 8m + 7.
template <typename T, int L, bool VEC>
__global__ void __launch_bounds__(kGatherWarps * 32) gather_kernel(const GatherParams P) {
    constexpr bool k8 = layout_fp8_keys(L), k3 = layout_3bit_keys(L), v3 = layout_3bit_values(L), aos = layout_is_aos(L);
    constexpr int nc = k3 ? 8 : kNumCentroids;
    constexpr int kKey = aos_key_bytes(L), kVal = val_code_bytes(L), kRow = kKey + kVal;  // SoA row
    __shared__ float scent[kNumCentroids];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, m = lane & 15;
    if constexpr (!k8) {
        if (threadIdx.x < nc) scent[threadIdx.x] = __ldg(P.cents + threadIdx.x);
        __syncthreads();
    }
    const uint32_t total = (uint32_t)P.N * (uint32_t)P.Hk;
    const uint32_t w0 = (blockIdx.x * kGatherWarps + (uint32_t)warp) * 2u;
    if (w0 >= total) return;
    const uint32_t pid0 = w0 + (uint32_t)(lane >> 4);
    const bool live = pid0 < total;
    const uint32_t pid = live ? pid0 : total - 1;
    const uint32_t n = pid / (uint32_t)P.Hk, h = pid - n * (uint32_t)P.Hk;
    const int32_t slot = __ldg(P.slots + n);
    const bool ok = slot >= 0 && (P.num_blocks <= 0 || (int64_t)slot < P.num_blocks * kBlockSize);
    const uint32_t blk = ok ? (uint32_t)slot / kBlockSize : 0u, off = ok ? (uint32_t)slot % kBlockSize : 0u;
    const uint8_t* base = P.cache + (size_t)blk * (size_t)P.block_bytes;
    const uint8_t *kp, *vp;
    float norm = 1.0f, scale, zero;
    if constexpr (aos) {
        const uint8_t* sp = base + (size_t)off * P.pos_stride + (size_t)h * P.head_stride;
        kp = sp;
        vp = sp + aos_val_off(L);
        if constexpr (!k8) norm = half_bits_to_float(ldu16(sp + aos_norm_off(L)));
        scale = half_bits_to_float(ldu16(sp + aos_scale_off(L)));
        zero = half_bits_to_float(ldu16(sp + aos_scale_off(L) + 2));
    } else {
        kp = base + (size_t)off * ((size_t)P.Hk * kRow) + (size_t)h * kRow;
        vp = kp + kKey;
        constexpr int kFields = k8 ? 2 : 3;
        const uint8_t* meta = base + (size_t)kBlockSize * P.Hk * kRow + ((size_t)h * kFields * kBlockSize + off) * 2;
        if constexpr (!k8) norm = half_bits_to_float(ldu16(meta));
        scale = half_bits_to_float(ldu16(meta + (kFields - 2) * kBlockSize * 2));
        zero = half_bits_to_float(ldu16(meta + (kFields - 1) * kBlockSize * 2));
    }
    float k[8], v[8];
    if constexpr (k8) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t h2 = fp8x2_to_h2(ldu16(kp + 8 * m + 2 * j));
            k[2 * j] = half_bits_to_float(h2);
            k[2 * j + 1] = half_bits_to_float(h2 >> 16);
        }
    } else {
        const uint32_t bits = k3 ? ld_bytes3(kp + 3 * m) : ldu16(kp + 4 * m) | (ldu16(kp + 4 * m + 2) << 16);
        float csq = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            k[j] = scent[(bits >> ((k3 ? 3 : 4) * j)) & (nc - 1)];
            csq = fmaf(k[j], k[j], csq);
        }
        // AoS stores |k|: the centroids are scaled to unit length here
        if constexpr (aos) norm = __fdiv_rn(norm, __fsqrt_rn(warp_sum_xor(csq, 1, 8) + 1e-16f));
#pragma unroll
        for (int j = 0; j < 8; j++) k[j] *= norm;
    }
    const uint32_t bits = v3 ? ld_bytes3(vp + 3 * m) : ldu16(vp + 4 * m) | (ldu16(vp + 4 * m + 2) << 16);
#pragma unroll
    for (int j = 0; j < 8; j++)
        v[j] = fmaf((float)((bits >> ((v3 ? 3 : 4) * j)) & (v3 ? 7u : 15u)), scale, zero);
    if (!live) return;
    if (!ok) {
#pragma unroll
        for (int j = 0; j < 8; j++) k[j] = v[j] = 0.0f;
    }
    put8<T, VEC>(static_cast<T*>(P.key) + (int64_t)n * P.ksn + (int64_t)h * P.ksh + 8 * m, k);
    put8<T, VEC>(static_cast<T*>(P.value) + (int64_t)n * P.vsn + (int64_t)h * P.vsh + 8 * m, v);
}

template <typename T, int L>
int launch_gather_t(const GatherParams& P, cudaStream_t stream) {
    constexpr int a = 16 / (int)sizeof(T);
    const bool vec = ((reinterpret_cast<uintptr_t>(P.key) | reinterpret_cast<uintptr_t>(P.value)) & 15) == 0 &&
                     P.ksn % a == 0 && P.ksh % a == 0 && P.vsn % a == 0 && P.vsh % a == 0;
    const unsigned grid = (unsigned)(((int64_t)P.N * P.Hk + 2 * kGatherWarps - 1) / (2 * kGatherWarps));
    if (vec)
        gather_kernel<T, L, true><<<grid, kGatherWarps * 32, 0, stream>>>(P);
    else
        gather_kernel<T, L, false><<<grid, kGatherWarps * 32, 0, stream>>>(P);
    return report_launch(cudaGetLastError());
}

template <typename T>
int launch_gather_d(const GatherParams& P, cudaStream_t stream) {
    switch (P.layout) {
        case TQB_LAYOUT_SOA: return launch_gather_t<T, TQB_LAYOUT_SOA>(P, stream);
        case TQB_LAYOUT_SOA_K8: return launch_gather_t<T, TQB_LAYOUT_SOA_K8>(P, stream);
        case TQB_LAYOUT_SOA_K3: return launch_gather_t<T, TQB_LAYOUT_SOA_K3>(P, stream);
        case TQB_LAYOUT_SOA_K3V3: return launch_gather_t<T, TQB_LAYOUT_SOA_K3V3>(P, stream);
        case TQB_LAYOUT_AOS: return launch_gather_t<T, TQB_LAYOUT_AOS>(P, stream);
        case TQB_LAYOUT_AOS_K8: return launch_gather_t<T, TQB_LAYOUT_AOS_K8>(P, stream);
        case TQB_LAYOUT_AOS_K3: return launch_gather_t<T, TQB_LAYOUT_AOS_K3>(P, stream);
        case TQB_LAYOUT_AOS_K3V3: return launch_gather_t<T, TQB_LAYOUT_AOS_K3V3>(P, stream);
        default: return TQB_ERR_INVALID_ARG;
    }
}

}  // namespace

int launch_gather(const GatherParams& P, cudaStream_t stream) {
    if (P.N == 0) return TQB_OK;
    switch (P.dtype) {
        case TQB_DTYPE_F32: return launch_gather_d<float>(P, stream);
        case TQB_DTYPE_F16: return launch_gather_d<__half>(P, stream);
        case TQB_DTYPE_BF16: return launch_gather_d<__nv_bfloat16>(P, stream);
        default: return TQB_ERR_INVALID_ARG;
    }
}

}  // namespace tqb
