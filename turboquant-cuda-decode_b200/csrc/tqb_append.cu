// tqb_append.cu — new tokens into the paged cache, from the projections' raw
// keys and values: rotary positions, norm, rotation and quantised store, with
// the queries of the same tokens rotated on the way.
//
// For every token n and KV head h (x = rope(key[n, h], position[n])):
//     y = x R / (|x| + 1e-8),  code_e = #{k : mid_k <= y_e},
//     stored norm = |x| / sqrt(sum_e c[code_e]^2 + 1e-16)  (SoA with norm
//     correction) or |x|, in fp16; values as tqb_store quantises them;
//     q_rot[n, h] = rope(query[n, h]) R in fp32.
// FP8 keys store x itself as e4m3, and their queries are not rotated.
//
// Nothing is rounded to the inputs' 16 bits on the way: x is the exact pair
// a c - b s rounded once to fp32 (error-free transformations), and the codes
// are those of exact arithmetic.  A coordinate whose fp32 value lies within
// kNear of a border, and a norm whose fp32 value lies within kNormNear of a
// border between two fp16 numbers, are computed again in 64 bits by the whole
// warp (about one row in fifteen), so the bytes written do not depend on the
// order of any sum.  kNear covers the fp32 sums: 128 products of a unit row
// and a unit column, each partial sum off by at most 2^-24 of its magnitude
// (<= 1 by Cauchy-Schwarz), 128 * 2^-24 = 2^-17 in all.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "tqb_common.cuh"
#include "tqb_internal.h"
#include "tqb_quant_row.cuh"

namespace tqb {

namespace {

constexpr float kNear = 0x1p-17f;
constexpr float kNormNear = 0x1p-19f;

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// a c + b s rounded once: the products' and the sum's rounding errors are
// formed exactly (FMA and two-sum) and added back.
__device__ __forceinline__ float pair_rn(float a, float c, float b, float s) {
    const float p = __fmul_rn(a, c), q = __fmul_rn(b, s);
    const float e = __fadd_rn(__fmaf_rn(a, c, -p), __fmaf_rn(b, s, -q));
    const float t = __fadd_rn(p, q), bb = __fsub_rn(t, p);
    const float err = __fadd_rn(__fsub_rn(p, __fsub_rn(t, bb)), __fsub_rn(q, bb));
    const float r = __fadd_rn(t, __fadd_rn(err, e));
    return isfinite(t) ? r : t;
}

// Position of token n; -1 when it is outside the table (or there are no
// rotary positions: 0).
__device__ __forceinline__ int position_of(const AppendParams& P, int n) {
    if (P.pos == nullptr) return 0;
    const long long p = P.pos_is_64 ? __ldg(static_cast<const long long*>(P.pos) + n)
                                    : (long long)__ldg(static_cast<const int*>(P.pos) + n);
    return p >= 0 && p < P.max_pos ? (int)p : -1;
}

// Partner dim, table index and sign of dim d under the rotary rule: out_d =
// x_d cos_j + sign x_partner sin_j.
struct RopeDim {
    int partner, j;
    float sign;
};
__device__ __forceinline__ RopeDim rope_dim(const AppendParams& P, int d) {
    RopeDim r;
    if (P.interleaved) {
        r.partner = d ^ 1;
        r.j = d >> 1;
        r.sign = (d & 1) ? 1.0f : -1.0f;
    } else {
        const int h = P.rotary >> 1;
        const bool low = d < h;
        r.partner = low ? d + h : d - h;
        r.j = low ? d : d - h;
        r.sign = low ? -1.0f : 1.0f;
    }
    return r;
}

// Dim d of a row after the rotary positions, fp32 and fp64.
template <typename T>
__device__ __forceinline__ float rope_f32(const AppendParams& P, const T* row, const float* cs, int d) {
    const float x = to_f32<T>(row[d]);
    if (d >= P.rotary) return x;
    const RopeDim r = rope_dim(P, d);
    return pair_rn(x, __ldg(cs + r.j), to_f32<T>(row[r.partner]), r.sign * __ldg(cs + (P.rotary >> 1) + r.j));
}
template <typename T>
__device__ __forceinline__ double rope_f64(const AppendParams& P, const T* row, const float* cs, int d) {
    const double x = (double)to_f32<T>(row[d]);
    if (d >= P.rotary) return x;
    const RopeDim r = rope_dim(P, d);
    return x * (double)__ldg(cs + r.j) +
           (double)(r.sign * to_f32<T>(row[r.partner])) * (double)__ldg(cs + (P.rotary >> 1) + r.j);
}

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// |x| of a key row in 64 bits (whole warp).
template <typename T>
__device__ __noinline__ double exact_norm(const AppendParams& P, const T* row, const float* cs, int lane) {
    double q = 0.0;
    for (int i = 0; i < 4; i++) {
        const double x = rope_f64<T>(P, row, cs, lane + 32 * i);
        q += x * x;
    }
    return sqrt(warp_sum_f64(q));
}
// Code of coordinate e of a key row in 64 bits (whole warp).
template <typename T>
__device__ __noinline__ int exact_code(const AppendParams& P, const T* row, const float* cs, int e, int nc, int lane) {
    double q = 0.0, z = 0.0;
    for (int i = 0; i < 4; i++) {
        const int d = lane + 32 * i;
        const double x = rope_f64<T>(P, row, cs, d);
        q += x * x;
        z += x * (double)__ldg(P.rot + d * kHeadDim + e);
    }
    q = warp_sum_f64(q);
    z = warp_sum_f64(z);
    const double y = z / (sqrt(q) + 1e-8);
    int c = 0;
    for (int k = 0; k < nc - 1; k++) c += y >= (double)__ldg(P.mids + k) ? 1 : 0;
    return c;
}

template <typename T>
__device__ __forceinline__ const float* table_row(const AppendParams& P, int pos) {
    return P.cos_sin + (int64_t)max(pos, 0) * P.cs_stride;
}

// Key codes, norm and values of token-heads from y's numerator, and their
// slots.  Half a warp per token-head (lane m of 16: dims 8m .. 8m + 7), the
// two halves of a warp on two rows; every lane calls it.  z: this lane's 8
// coordinates of x R; nsq: the row's sum of x^2; x8: this lane's x (FP8 keys).
template <typename T, int L>
__device__ __forceinline__ void finish_row(const AppendParams& P, const float* smid, const float* scent, int n, int h,
                                           bool live, int lane, const float (&z)[8], float nsq) {
    constexpr bool k8 = layout_fp8_keys(L), k3 = layout_3bit_keys(L), v3 = layout_3bit_values(L);
    constexpr int nc = k3 ? 8 : kNumCentroids, kBits = k3 ? 3 : 4;
    constexpr unsigned kFull = 0xffffffffu;
    const int m = lane & 15;
    const T* krow = static_cast<const T*>(P.key) + (int64_t)n * P.ksn + (int64_t)h * P.ksh;
    const T* vrow = static_cast<const T*>(P.value) + (int64_t)n * P.vsn + (int64_t)h * P.vsh;
    const int pos = position_of(P, n);
    const float* cs = table_row<T>(P, pos);
    const int32_t slot = __ldg(P.slots + n);
    const bool write = live && pos >= 0 && slot >= 0 &&
                       (P.num_blocks <= 0 || (int64_t)slot < P.num_blocks * kBlockSize);
    uint32_t klo = 0, khi = 0, kbits = 0;
    unsigned short vn_h = 0;
    if constexpr (k8) {
        auto cvt2 = [](float a, float b) {
            return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
        };
        klo = cvt2(z[0], z[1]) | (cvt2(z[2], z[3]) << 16);
        khi = cvt2(z[4], z[5]) | (cvt2(z[6], z[7]) << 16);
    } else {
        const float norm = __fsqrt_rn(nsq), inv = __frcp_rn(norm + 1e-8f);
        int code[8];
        uint32_t near = 0;  // coordinates next to a border
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float y = z[j] * inv;
            int i;
            if constexpr (k3) {
                i = y >= smid[3] ? 4 : 0;
            } else {
                i = y >= smid[7] ? 8 : 0;
                i += y >= smid[i + 3] ? 4 : 0;
            }
            i += y >= smid[i + 1] ? 2 : 0;
            i += y >= smid[i] ? 1 : 0;
            code[j] = i;
            // the borders on the two sides of the code (one side at the ends)
            near |= (fabsf(y - smid[max(i - 1, 0)]) < kNear || fabsf(y - smid[min(i, nc - 2)]) < kNear) ? 1u << j : 0u;
        }
        if (!write) near = 0;
        uint32_t who;
        while ((who = __ballot_sync(kFull, near != 0)) != 0) {
            const int src = __ffs(who) - 1;
            const int sn = __shfl_sync(kFull, n, src), sh = __shfl_sync(kFull, h, src), sp = __shfl_sync(kFull, pos, src);
            const int j = __shfl_sync(kFull, __ffs(near) - 1, src);
            const T* row = static_cast<const T*>(P.key) + (int64_t)sn * P.ksn + (int64_t)sh * P.ksh;
            const int c = exact_code<T>(P, row, table_row<T>(P, sp), 8 * (src & 15) + j, nc, lane);
            if (lane == src) {
#pragma unroll
                for (int jj = 0; jj < 8; jj++)
                    if (jj == j) code[jj] = c;
                near &= near - 1;
            }
        }
        float csq = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            kbits |= (uint32_t)code[j] << (kBits * j);
            const float c = scent[code[j]];
            csq = fmaf(c, c, csq);
        }
        float stored = norm;
        const bool fold = !layout_is_aos(L) && P.norm_correction;
        if (fold) stored = norm * rsqrtf(warp_sum_xor(csq, 1, 8) + 1e-16f);
        vn_h = __half_as_ushort(__float2half_rn(stored));
        const bool split = __half_as_ushort(__float2half_rn(stored * (1.0f - kNormNear))) !=
                           __half_as_ushort(__float2half_rn(stored * (1.0f + kNormNear)));
        uint32_t ask = __ballot_sync(kFull, m == 0 && write && split);
        while (ask != 0) {
            const int src = __ffs(ask) - 1;
            ask &= ask - 1;
            const int sn = __shfl_sync(kFull, n, src), sh = __shfl_sync(kFull, h, src), sp = __shfl_sync(kFull, pos, src);
            const T* row = static_cast<const T*>(P.key) + (int64_t)sn * P.ksn + (int64_t)sh * P.ksh;
            double v = exact_norm<T>(P, row, table_row<T>(P, sp), lane);
            double cq = 0.0;
            if (fold && (lane & 16) == (src & 16)) {
#pragma unroll
                for (int j = 0; j < 8; j++) cq += (double)scent[code[j]] * (double)scent[code[j]];
            }
            cq = warp_sum_f64(cq);
            if (fold) v /= sqrt(cq + 1e-16);
            if (lane == src) vn_h = __half_as_ushort(__double2half(v));
        }
    }
    float vs[8];
#pragma unroll
    for (int j = 0; j < 8; j++) vs[j] = to_f32<T>(vrow[8 * m + j]);
    const ValueRow vr = quantise_values<v3>(vs);
    if (!write) return;
    write_row<L>(P.cache + (size_t)((uint32_t)slot / kBlockSize) * (size_t)P.block_bytes, (uint32_t)slot % kBlockSize,
                 (uint32_t)h, P.Hk, P.pos_stride, P.head_stride, m, kbits, klo, khi, vr.bits, vn_h, vr.scale, vr.vmin);
}

// ---------------------------------------------------------------------------
// Any alignment and strides: a CTA takes 32 rows (of keys, then of queries),
// forms x in shared memory, multiplies by R (64 KB, staged) with fp32 FMAs,
// and finishes key rows half a warp each.
// ---------------------------------------------------------------------------
constexpr int kRows = 32;
constexpr int kAppThreads = 256;
constexpr int kAppSmem = (kHeadDim * kHeadDim + kRows * kHeadDim) * 4;

template <typename T, int L>
__global__ void __launch_bounds__(kAppThreads) append_kernel(const AppendParams P, int key_ctas) {
    constexpr bool k8 = layout_fp8_keys(L), k3 = layout_3bit_keys(L);
    constexpr int nc = k3 ? 8 : kNumCentroids;
    extern __shared__ __align__(16) float asm_[];
    __shared__ float smid[kNumCentroids], scent[kNumCentroids];
    float* xs = asm_;                        // [kRows][128]
    float* Rs = asm_ + kRows * kHeadDim;     // [128][128] (not for FP8 keys)
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const bool keys = (int)blockIdx.x < key_ctas;
    const int H = keys ? P.Hk : P.Hq;
    const uint32_t total = (uint32_t)P.N * (uint32_t)H;
    const uint32_t r0 = ((uint32_t)blockIdx.x - (keys ? 0u : (uint32_t)key_ctas)) * kRows;
    if constexpr (!k8) {
        if (t < nc - 1) smid[t] = __ldg(P.mids + t);
        if (t < nc) scent[t] = __ldg(P.cents + t);
        const float4* R4 = reinterpret_cast<const float4*>(P.rot);
        for (int e = t; e < kHeadDim * kHeadDim / 4; e += kAppThreads) reinterpret_cast<float4*>(Rs)[e] = __ldg(R4 + e);
    }
    const T* base = static_cast<const T*>(keys ? P.key : P.query);
    const int64_t sn = keys ? P.ksn : P.qsn, sh = keys ? P.ksh : P.qsh;
    const int d = t % kHeadDim;
    for (int i = t / kHeadDim; i < kRows; i += kAppThreads / kHeadDim) {
        float x = 0.0f;
        if (r0 + i < total) {
            const uint32_t n = (r0 + i) / (uint32_t)H, h = (r0 + i) - n * (uint32_t)H;
            const int pos = position_of(P, (int)n);
            // a query whose position is outside the table has no value
            x = pos < 0 && !keys ? __int_as_float(0x7fc00000)
                                 : rope_f32<T>(P, base + (int64_t)n * sn + (int64_t)h * sh, table_row<T>(P, pos), d);
        }
        xs[i * kHeadDim + d] = x;
    }
    __syncthreads();
    float nsq[2];  // sums of squares of this half-warp's two rows
    const int m = lane & 15, half = (lane >> 4) + 2 * warp;
    if (keys) {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const float* x = xs + (half + 16 * k) * kHeadDim + 8 * m;
            float q = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) q = fmaf(x[j], x[j], q);
            nsq[k] = warp_sum_xor(q, 1, 8);
        }
    }
    if constexpr (!k8) {
        constexpr int kPer = kRows / (kAppThreads / kHeadDim);  // rows per thread
        const int i0 = (t / kHeadDim) * kPer;
        float acc[kPer];
#pragma unroll
        for (int i = 0; i < kPer; i++) acc[i] = 0.0f;
#pragma unroll 2
        for (int k = 0; k < kHeadDim; k += 4) {
            const float a = Rs[k * kHeadDim + d], b = Rs[(k + 1) * kHeadDim + d], c = Rs[(k + 2) * kHeadDim + d],
                        e = Rs[(k + 3) * kHeadDim + d];
#pragma unroll
            for (int i = 0; i < kPer; i++) {
                const float4 x = *reinterpret_cast<const float4*>(xs + (i0 + i) * kHeadDim + k);
                acc[i] = fmaf(x.w, e, fmaf(x.z, c, fmaf(x.y, b, fmaf(x.x, a, acc[i]))));
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kPer; i++) xs[(i0 + i) * kHeadDim + d] = acc[i];
        __syncthreads();
    }
    if (!keys) {
        for (int i = t / kHeadDim; i < kRows; i += kAppThreads / kHeadDim) {
            if (r0 + i >= total) break;
            const uint32_t n = (r0 + i) / (uint32_t)H, h = (r0 + i) - n * (uint32_t)H;
            P.q_rot[(int64_t)n * P.osn + (int64_t)h * P.osh + d] = xs[i * kHeadDim + d];
        }
        return;
    }
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const uint32_t row = r0 + half + 16 * k;
        const bool live = row < total;
        const uint32_t rc = live ? row : total - 1;
        const uint32_t n = rc / (uint32_t)H, h = rc - n * (uint32_t)H;
        float z[8];
#pragma unroll
        for (int j = 0; j < 8; j++) z[j] = xs[(half + 16 * k) * kHeadDim + 8 * m + j];
        finish_row<T, L>(P, smid, scent, (int)n, (int)h, live, lane, z, nsq[k]);
    }
}

template <typename T, int L>
int launch_append_t(const AppendParams& P, cudaStream_t stream) {
    auto kern = append_kernel<T, L>;
    const int smem = layout_fp8_keys(L) ? kRows * kHeadDim * 4 : kAppSmem;
    static thread_local int configured_dev = -1;
    int dev = 0;
    cudaGetDevice(&dev);
    if (configured_dev != dev) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
            return report_launch(cudaGetLastError());
        configured_dev = dev;
    }
    const int64_t kc = ((int64_t)P.N * P.Hk + kRows - 1) / kRows;
    const int64_t qc = P.query ? ((int64_t)P.N * P.Hq + kRows - 1) / kRows : 0;
    kern<<<(unsigned)(kc + qc), kAppThreads, smem, stream>>>(P, (int)kc);
    return report_launch(cudaGetLastError());
}

template <typename T>
int launch_append_d(const AppendParams& P, cudaStream_t stream) {
    switch (P.layout) {
        case TQB_LAYOUT_SOA: return launch_append_t<T, TQB_LAYOUT_SOA>(P, stream);
        case TQB_LAYOUT_SOA_K8: return launch_append_t<T, TQB_LAYOUT_SOA_K8>(P, stream);
        case TQB_LAYOUT_SOA_K3: return launch_append_t<T, TQB_LAYOUT_SOA_K3>(P, stream);
        case TQB_LAYOUT_SOA_K3V3: return launch_append_t<T, TQB_LAYOUT_SOA_K3V3>(P, stream);
        case TQB_LAYOUT_AOS: return launch_append_t<T, TQB_LAYOUT_AOS>(P, stream);
        case TQB_LAYOUT_AOS_K8: return launch_append_t<T, TQB_LAYOUT_AOS_K8>(P, stream);
        case TQB_LAYOUT_AOS_K3: return launch_append_t<T, TQB_LAYOUT_AOS_K3>(P, stream);
        case TQB_LAYOUT_AOS_K3V3: return launch_append_t<T, TQB_LAYOUT_AOS_K3V3>(P, stream);
        default: return TQB_ERR_INVALID_ARG;
    }
}

}  // namespace

int launch_append(const AppendParams& P, cudaStream_t stream, int num_sms) {
    (void)num_sms;
    if (P.N == 0) return TQB_OK;
    switch (P.dtype) {
        case TQB_DTYPE_F32: return launch_append_d<float>(P, stream);
        case TQB_DTYPE_F16: return launch_append_d<__half>(P, stream);
        case TQB_DTYPE_BF16: return launch_append_d<__nv_bfloat16>(P, stream);
        default: return TQB_ERR_INVALID_ARG;
    }
}

}  // namespace tqb
