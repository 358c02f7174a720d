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
// with 16-bit outputs, so HBM writes bound it.  131072 tokens of 8 heads: 127 us,
// 5.3 TB/s.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "tqb_common.cuh"
#include "tqb_internal.h"

namespace tqb {

namespace {

constexpr int kGatherWarps = 8, kIn = 2;

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

// What half a warp reads of a token-head: lane m of 16 takes dims 8m .. 8m + 7.
template <int L>
struct Row {
    uint32_t n, h, k[layout_fp8_keys(L) ? 2 : 1], v, norm, scale, zero;
    bool ok;
};

// A4: codes at 4-byte aligned addresses.
template <int L, bool A4>
__device__ __forceinline__ uint32_t codes8(const uint8_t* p, int m, bool three) {
    if (three) return ld_bytes3(p + 3 * m);
    if constexpr (A4) return __ldg(reinterpret_cast<const uint32_t*>(p + 4 * m));
    return ldu16(p + 4 * m) | (ldu16(p + 4 * m + 2) << 16);
}

template <int L, bool A4>
__device__ __forceinline__ void load_row(Row<L>& r, const GatherParams& P, uint32_t pid, int m) {
    constexpr bool k8 = layout_fp8_keys(L), k3 = layout_3bit_keys(L), v3 = layout_3bit_values(L), aos = layout_is_aos(L);
    constexpr int kKey = aos_key_bytes(L), kVal = val_code_bytes(L), kRow = kKey + kVal;  // SoA row
    r.n = P.div_hk.div(pid);
    r.h = pid - r.n * (uint32_t)P.Hk;
    const int32_t slot = __ldg(P.slots + r.n);
    r.ok = slot >= 0 && (P.num_blocks <= 0 || (int64_t)slot < P.num_blocks * kBlockSize);
    const uint32_t blk = r.ok ? (uint32_t)slot / kBlockSize : 0u, off = r.ok ? (uint32_t)slot % kBlockSize : 0u;
    const uint8_t* base = P.cache + (size_t)blk * (size_t)P.block_bytes;
    const uint8_t *kp, *vp;
    if constexpr (aos) {
        kp = base + (size_t)off * P.pos_stride + (size_t)r.h * P.head_stride;
        vp = kp + aos_val_off(L);
        if constexpr (!k8) r.norm = ldu16(kp + aos_norm_off(L));
        r.scale = ldu16(kp + aos_scale_off(L));
        r.zero = ldu16(kp + aos_scale_off(L) + 2);
    } else {
        kp = base + (size_t)off * ((size_t)P.Hk * kRow) + (size_t)r.h * kRow;
        vp = kp + kKey;
        constexpr int kFields = k8 ? 2 : 3;
        const uint8_t* meta = base + (size_t)kBlockSize * P.Hk * kRow + ((size_t)r.h * kFields * kBlockSize + off) * 2;
        if constexpr (!k8) r.norm = ldu16(meta);
        r.scale = ldu16(meta + (kFields - 2) * kBlockSize * 2);
        r.zero = ldu16(meta + (kFields - 1) * kBlockSize * 2);
    }
    if constexpr (k8) {
        r.k[0] = codes8<L, A4>(kp, 2 * m, false);
        r.k[1] = codes8<L, A4>(kp, 2 * m + 1, false);
    } else {
        r.k[0] = codes8<L, A4>(kp, m, k3);
    }
    r.v = codes8<L, A4>(vp, m, v3);
}

// kIn token-heads per half-warp, all their loads in flight together; the
// codebook in shared memory as pairs, so that a table entry is two numbers.
// (kIn = 1, with single numbers: 141 us; 2: 127; 4: 125, but 917 tokens of 2
// heads take 3.1 us in place of 2.4; 8: 144.)
template <typename T, int L, bool VEC, bool A4>
__global__ void __launch_bounds__(kGatherWarps * 32) gather_kernel(const __grid_constant__ GatherParams P) {
    constexpr bool k8 = layout_fp8_keys(L), k3 = layout_3bit_keys(L), v3 = layout_3bit_values(L), aos = layout_is_aos(L);
    constexpr int kb = k3 ? 3 : 4, nc = 1 << kb;
    __shared__ float2 pairs[nc * nc];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, m = lane & 15;
    const uint32_t total = (uint32_t)P.N * (uint32_t)P.Hk;
    const uint32_t w0 = (blockIdx.x * kGatherWarps + (uint32_t)warp) * (2u * kIn) + (uint32_t)(lane >> 4);
    Row<L> row[kIn];
#pragma unroll
    for (int i = 0; i < kIn; i++) load_row<L, A4>(row[i], P, min(w0 + 2u * i, total - 1), m);
    if constexpr (!k8) {
        if (threadIdx.x < nc * nc) pairs[threadIdx.x] = make_float2(__ldg(P.cents + threadIdx.x % nc), __ldg(P.cents + threadIdx.x / nc));
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < kIn; i++) {
        const Row<L>& r = row[i];
        float k[8], v[8];
        if constexpr (k8) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t h2 = fp8x2_to_h2((r.k[j >> 1] >> (16 * (j & 1))) & 0xffffu);
                k[2 * j] = half_bits_to_float(h2);
                k[2 * j + 1] = half_bits_to_float(h2 >> 16);
            }
        } else {
            float norm = half_bits_to_float(r.norm), csq = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 c = pairs[(r.k[0] >> (2 * kb * j)) & (nc * nc - 1)];
                k[2 * j] = c.x;
                k[2 * j + 1] = c.y;
                if constexpr (aos) csq = fmaf(c.y, c.y, fmaf(c.x, c.x, csq));
            }
            // AoS stores |k|: the centroids are scaled to unit length here
            if constexpr (aos) norm = __fdiv_rn(norm, __fsqrt_rn(warp_sum_xor(csq, 1, 8) + 1e-16f));
#pragma unroll
            for (int j = 0; j < 8; j++) k[j] *= norm;
        }
        const float scale = half_bits_to_float(r.scale), zero = half_bits_to_float(r.zero);
#pragma unroll
        for (int j = 0; j < 8; j++)
            v[j] = fmaf((float)((r.v >> ((v3 ? 3 : 4) * j)) & (v3 ? 7u : 15u)), scale, zero);
        if (!r.ok) {
#pragma unroll
            for (int j = 0; j < 8; j++) k[j] = v[j] = 0.0f;
        }
        if (w0 + 2u * i >= total) continue;
        put8<T, VEC>(static_cast<T*>(P.key) + (int64_t)r.n * P.ksn + (int64_t)r.h * P.ksh + 8 * m, k);
        put8<T, VEC>(static_cast<T*>(P.value) + (int64_t)r.n * P.vsn + (int64_t)r.h * P.vsh + 8 * m, v);
    }
}

template <typename T, int L>
int launch_gather_t(const GatherParams& P, cudaStream_t stream) {
    constexpr int a = 16 / (int)sizeof(T);
    const bool vec = ((reinterpret_cast<uintptr_t>(P.key) | reinterpret_cast<uintptr_t>(P.value)) & 15) == 0 &&
                     P.ksn % a == 0 && P.ksh % a == 0 && P.vsn % a == 0 && P.vsh % a == 0;
    const bool a4 = ((reinterpret_cast<uintptr_t>(P.cache) | (uintptr_t)P.block_bytes) & 3) == 0 && !layout_is_aos(L);
    constexpr int kRows = 2 * kIn * kGatherWarps;
    const unsigned grid = (unsigned)(((int64_t)P.N * P.Hk + kRows - 1) / kRows);
    auto kern = vec ? (a4 ? gather_kernel<T, L, true, true> : gather_kernel<T, L, true, false>) : gather_kernel<T, L, false, false>;
    kern<<<grid, kGatherWarps * 32, 0, stream>>>(P);
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
