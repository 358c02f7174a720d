// tqb_store.cu — sm_100a TurboQuant cache store (all presets, SoA and AoS).
//
// Reference: _tq_fused_store_mse in reference/soa_store.py:223-373 (SoA) and
// reference/aos_store.py:221-340 (AoS).  Half a warp per token-head, each
// lane owning 8 consecutive dims, one kernel instance per layout:
//   1. bucketise y (rotated unit key) against the 15 midpoints with the
//      reference's 4-step binary search, `y >= mid` going right (:306-316);
//   2. pack two codes per byte, low nibble = even dim (:319-325);
//   3. SoA with norm correction: stored norm = fp16(|k| * (1/sqrt(sum c^2 +
//      1e-16))) (:343-353); AoS: fp16(|k|);
//   4. values: min/max, scale = max((max-min)/15, 1e-8), code =
//      clamp(trunc((v-min)/scale + 0.5), 0, 15), fp16 scale and zero (:85-116).
// All fp32 steps use explicitly rounded intrinsics, and the 128-term sum of
// squared centroids follows the reference's summation order (eight strided
// running sums combined pairwise, the order numpy applies when the reference
// kernel runs interpreted), so the written bytes are bit-identical to the
// reference store for the same kernel inputs.
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "tqb_common.cuh"
#include "tqb_internal.h"
#include "tqb_quant_row.cuh"

namespace tqb {

namespace {

constexpr int kStoreWarps = 8;

// One instance per cache layout L, so each carries only its own key and
// slot code.  A token-head takes 16 lanes, 8 consecutive dims per lane
// (dims 8m .. 8m + 7 on lane m of the half-warp), so a warp stores two
// token-heads and the per-row reductions are 4 shuffle levels.  The
// midpoints and the squared centroids sit in shared memory.
template <int L>
__global__ void __launch_bounds__(kStoreWarps * 32) store_kernel(const StoreParams P) {
    constexpr bool k8 = layout_fp8_keys(L), k3 = layout_3bit_keys(L), v3 = layout_3bit_values(L);
    constexpr int nc = k3 ? 8 : kNumCentroids;
    constexpr unsigned kFull = 0xffffffffu;
    __shared__ float4 sq[2 * kStoreWarps][kHeadDim / 4];  // squared centroids of each row
    __shared__ float smid[kNumCentroids], scsq[kNumCentroids];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, m = lane & 15, half = lane >> 4;
    if constexpr (!k8) {
        if (threadIdx.x < nc - 1) smid[threadIdx.x] = __ldg(P.mids + threadIdx.x);
        if (P.norm_correction && threadIdx.x < nc) {
            const float cv = __ldg(P.cents + threadIdx.x);
            scsq[threadIdx.x] = __fmul_rn(cv, cv);
        }
        __syncthreads();
    }
    // N x H < 2^31 (checked on the host): 32-bit index arithmetic.  A warp
    // past the end leaves as a whole; a half past the end, or on a padding
    // token, computes on the last row and stores nothing, so every shuffle
    // runs on all 32 lanes.
    const uint32_t total = (uint32_t)P.N * (uint32_t)P.H;
    const uint32_t w0 = (blockIdx.x * kStoreWarps + (uint32_t)warp) * 2u;
    if (w0 >= total) return;
    const uint32_t pid0 = w0 + (uint32_t)half;
    const bool live = pid0 < total;
    const uint32_t pid = live ? pid0 : total - 1;
    const uint32_t tok = pid / (uint32_t)P.H, h = pid - tok * (uint32_t)P.H;
    const int32_t slot = __ldg(P.slots + tok);
    const bool write = live && slot >= 0;  // slot < 0: padding token (reference/soa_store.py:275-277)
    const uint32_t blk = (uint32_t)max(slot, 0) / kBlockSize, off = (uint32_t)max(slot, 0) % kBlockSize;

    const float4* yp = reinterpret_cast<const float4*>(P.y + (size_t)pid * kHeadDim) + 2 * m;
    const float4* vp4 = reinterpret_cast<const float4*>(P.value + (size_t)pid * kHeadDim) + 2 * m;
    const float4 ya = __ldg(yp), yb = __ldg(yp + 1), va = __ldg(vp4), vb = __ldg(vp4 + 1);
    uint32_t klo = 0, khi = 0;  // key codes: dims 8m .. 8m+3 in klo, 8m+4 .. 8m+7 in khi (FP8: bytes)
    uint32_t kbits = 0;         // 4-bit: 8 nibbles; 3-bit: 24 bits
    float vn = 0.0f;
    if constexpr (k8) {
        // FP8 keys (reference/soa_store.py:187-194): the raw key cast to e4m3
        // with round-to-nearest-even and saturation to +-448, the conversion
        // the compiled reference issues on sm_90 and later.
        auto cvt2 = [](float a, float b) {
            return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
        };
        klo = cvt2(ya.x, ya.y) | (cvt2(ya.z, ya.w) << 16);
        khi = cvt2(yb.x, yb.y) | (cvt2(yb.z, yb.w) << 16);
    } else {
        // -- keys: bucketise + pack.  The reference's binary search
        // (reference/soa_store.py:305-316; `y >= mid` goes right, 4 steps, or
        // 3 for 8 centroids) visits the midpoints of a complete binary tree:
        // 7, then 3 or 11, then idx + 1, then idx (3-bit: 3, idx + 1, idx),
        // never reaching the clamp at nc - 2, so this walk is the same search.
        vn = __ldg(P.norms + pid);
        const float ys[8] = {ya.x, ya.y, ya.z, ya.w, yb.x, yb.y, yb.z, yb.w};
        int idx[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            int i;
            if constexpr (k3) {
                i = ys[j] >= smid[3] ? 4 : 0;
            } else {
                i = ys[j] >= smid[7] ? 8 : 0;
                i += ys[j] >= smid[i + 3] ? 4 : 0;
            }
            i += ys[j] >= smid[i + 1] ? 2 : 0;
            i += ys[j] >= smid[i] ? 1 : 0;
            idx[j] = i;
            kbits |= (uint32_t)i << ((k3 ? 3 : 4) * j);
        }

        if (P.norm_correction) {
            // 8 strided running sums r_i = c^2[i] + c^2[i+8] + ... + c^2[i+120]
            // in that order (the row's lanes m = 0..15 in turn), then
            // ((r0 + r1) + (r2 + r3)) + ((r4 + r5) + (r6 + r7))
            float4* row = sq[2 * warp + half];
            row[2 * m] = make_float4(scsq[idx[0]], scsq[idx[1]], scsq[idx[2]], scsq[idx[3]]);
            row[2 * m + 1] = make_float4(scsq[idx[4]], scsq[idx[5]], scsq[idx[6]], scsq[idx[7]]);
            __syncwarp();
            const float* rs = reinterpret_cast<const float*>(row) + (m & 7);
            float r = rs[0];
#pragma unroll
            for (int k = 1; k < 16; k++) r = __fadd_rn(r, rs[8 * k]);  // r_{m & 7}
            const float r1 = __shfl_down_sync(kFull, r, 1);
            const float pr = __fadd_rn(r, r1);  // valid on even m < 8
            const float pr2 = __shfl_down_sync(kFull, pr, 2);
            const float qd = __fadd_rn(pr, pr2);  // valid on m = 0, 4
            const float qd4 = __shfl_down_sync(kFull, qd, 4);
            float nsq = __fadd_rn(qd, qd4);  // valid on m = 0
            nsq = __shfl_sync(kFull, nsq, lane & 16);
            nsq = __fadd_rn(nsq, 1e-16f);
            vn = __fmul_rn(vn, __frcp_rn(__fsqrt_rn(nsq)));  // RN(1/x) = RN(1 / x)
        }
    }

    // -- values: quantise + pack --
    const float vs[8] = {va.x, va.y, va.z, va.w, vb.x, vb.y, vb.z, vb.w};
    const ValueRow vr = quantise_values<v3>(vs);
    if (!write) return;

    // -- write --
    // AoS stores the raw norm (its decoders apply the correction)
    if constexpr (layout_is_aos(L) && !k8) vn = __ldg(P.norms + pid);
    write_row<L>(P.cache + (size_t)blk * (size_t)P.block_bytes, off, h, P.H, P.pos_stride, P.head_stride, m, kbits, klo,
                 khi, vr, __half_as_ushort(__float2half_rn(vn)));
}

}  // namespace

template <int L>
void launch_store_t(const StoreParams& P, unsigned grid, cudaStream_t stream) {
    store_kernel<L><<<grid, kStoreWarps * 32, 0, stream>>>(P);
}

int launch_store(const StoreParams& P, cudaStream_t stream) {
    const int64_t items = (int64_t)P.N * P.H;
    if (items == 0) return TQB_OK;
    const unsigned grid = (unsigned)((items + 2 * kStoreWarps - 1) / (2 * kStoreWarps));
    switch (P.layout) {
        case TQB_LAYOUT_SOA: launch_store_t<TQB_LAYOUT_SOA>(P, grid, stream); break;
        case TQB_LAYOUT_SOA_K8: launch_store_t<TQB_LAYOUT_SOA_K8>(P, grid, stream); break;
        case TQB_LAYOUT_SOA_K3: launch_store_t<TQB_LAYOUT_SOA_K3>(P, grid, stream); break;
        case TQB_LAYOUT_SOA_K3V3: launch_store_t<TQB_LAYOUT_SOA_K3V3>(P, grid, stream); break;
        case TQB_LAYOUT_AOS: launch_store_t<TQB_LAYOUT_AOS>(P, grid, stream); break;
        case TQB_LAYOUT_AOS_K8: launch_store_t<TQB_LAYOUT_AOS_K8>(P, grid, stream); break;
        case TQB_LAYOUT_AOS_K3: launch_store_t<TQB_LAYOUT_AOS_K3>(P, grid, stream); break;
        case TQB_LAYOUT_AOS_K3V3: launch_store_t<TQB_LAYOUT_AOS_K3V3>(P, grid, stream); break;
        default: return TQB_ERR_INVALID_ARG;
    }
    return report_launch(cudaGetLastError());
}

}  // namespace tqb
