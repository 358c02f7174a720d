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
// Nothing is rounded to the inputs' 16 bits on the way, and the codes are those
// of exact arithmetic.  A coordinate whose fp32 value lies within kNear of a
// border, and a norm whose fp32 value lies within kNormNear (relative) of a
// border between two fp16 numbers, are computed again in 64 bits by the whole
// warp (about one row in forty, and one in two hundred), so the bytes written do
// not depend on the order of any sum.  Bounds, in units of 2^-23, the larger of
// the two forms below:
//   y (of |x|; partial sums of a unit row times a unit column stay below 1,
//   Cauchy-Schwarz): the turned pairs 1; the splits of x and R 2 each and the
//   product of the two rests 2; eight accumulations of the full-size products 8
//   (the others are 2^-8 of them or less); the norm and its reciprocal, as
//   below without c, 6; the border in the cell table, whose four low bits hold
//   its index, 2 (15 units of 2^-26).  23 in all, kNear is 24.
//   (Measured, largest of 65536 rows along a column of R, where every partial
//   sum is near 1: 2^-19.9 with tcgen05, 2^-21.4 with mma.sync; of random rows
//   2^-22.5 and 2^-23.4.)
//   stored norm: the turned pairs 1; |x|^2 in a chain of 8 and 4 additions,
//   halved by the root, 3; the root 0.5; sum c^2 in chains of 16 and 8
//   additions, its squares rounded, halved, 6; rsqrtf 2, the product 0.5.  13
//   in all, kNormNear is 16.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "tqb_common.cuh"
#include "tqb_internal.h"
#include "tqb_quant_row.cuh"
#include "tqb_rot_mma.cuh"
#include "tqb_umma.cuh"

namespace tqb {

// Kernels that gave up a wait (read by tqb_wait_timeouts).
__device__ unsigned int g_append_timeouts = 0;

namespace {

constexpr float kNear = 24 * 0x1p-23f;
constexpr float kNormNear = 16 * 0x1p-23f;

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
// Code of coordinate e of a key row in 64 bits (whole warp): the borders with
// x R_e >= mid (|x| + 1e-8), a lane each (borders may lie closer to one another
// than fp32 can tell).
template <typename T>
__device__ __noinline__ int exact_code(const AppendParams& P, const T* row, const float* cs, int e, const float* smid, int borders,
                                       int lane) {
    double q = 0.0, z = 0.0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int d = lane + 32 * i;
        const double x = rope_f64<T>(P, row, cs, d);
        q += x * x;
        z += x * (double)__ldg(P.rot + d * kHeadDim + e);
    }
    q = warp_sum_f64(q);
    z = warp_sum_f64(z);
    return __popc(__ballot_sync(0xffffffffu, lane < borders && z >= (double)smid[min(lane, borders - 1)] * (sqrt(q) + 1e-8)));
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
            const float below = fabsf(y - smid[max(i - 1, 0)]), above = fabsf(y - smid[min(i, nc - 2)]);
            near |= fminf(below, above) < kNear ? 1u << j : 0u;
        }
        if (__any_sync(kFull, nsq == 0.0f)) {
            // a row of zeros has its coordinates at 0 exactly, next to a middle
            // border all of them: no 64 bits for it (its elements are asked, as
            // the squares of small ones vanish too)
            bool some = false;
#pragma unroll
            for (int j = 0; j < 8; j++) some |= to_f32<T>(krow[8 * m + j]) != 0.0f;
            const uint32_t rows = __ballot_sync(kFull, some);
            if (nsq == 0.0f && ((rows >> (lane & 16)) & 0xFFFFu) == 0) near = 0;
        }
        if (!(norm < INFINITY)) {  // a stored norm of inf or NaN: no codes
            near = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) code[j] = 0;
        }
        if (!write) near = 0;
        uint32_t who;
        while ((who = __ballot_sync(kFull, near != 0)) != 0) {
            const int src = __ffs(who) - 1;
            const int sn = __shfl_sync(kFull, n, src), sh = __shfl_sync(kFull, h, src), sp = __shfl_sync(kFull, pos, src);
            const int j = __shfl_sync(kFull, __ffs(near) - 1, src);
            const T* row = static_cast<const T*>(P.key) + (int64_t)sn * P.ksn + (int64_t)sh * P.ksh;
            const int c = exact_code<T>(P, row, table_row<T>(P, sp), 8 * (src & 15) + j, smid, nc - 1, lane);
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
                 (uint32_t)h, P.Hk, P.pos_stride, P.head_stride, m, kbits, klo, khi, vr, vn_h);
}

// ---------------------------------------------------------------------------
// Few rows, or inputs of any alignment, and the FP8-key layouts: a CTA of four
// warps takes 16 rows (of keys, then of queries), turns them into shared
// memory, multiplies by R on the register-operand tensor cores (rot_step: the
// rows in three parts) and finishes key rows half a warp each.  R's fragments
// come from L2, so that nothing has to be staged before the first product: the
// latency of a decode step's call counts here.
// ---------------------------------------------------------------------------
constexpr int kRows = 16;
constexpr int kAppThreads = 128;
constexpr int kPitch = kHeadDim + 16;  // floats of a row in shared memory: a pair of rows covers the 32 banks

template <typename T, int L>
__global__ void __launch_bounds__(kAppThreads) append_kernel(const __grid_constant__ AppendParams P, int key_ctas) {
    constexpr bool k8 = layout_fp8_keys(L), k3 = layout_3bit_keys(L);
    constexpr int nc = k3 ? 8 : kNumCentroids;
    __shared__ __align__(16) float xs[kRows * kPitch];
    __shared__ float smid[kNumCentroids], scent[kNumCentroids];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const bool keys = (int)blockIdx.x < key_ctas;
    const uint32_t H = (uint32_t)(keys ? P.Hk : P.Hq);
    const FastDiv& div = keys ? P.div_hk : P.div_hq;
    const uint32_t total = (uint32_t)P.N * H;
    const uint32_t r0 = ((uint32_t)blockIdx.x - (keys ? 0u : (uint32_t)key_ctas)) * kRows;
    const T* base = static_cast<const T*>(keys ? P.key : P.query);
    const int64_t sn = keys ? P.ksn : P.qsn, sh = keys ? P.ksh : P.qsh;
    if constexpr (!k8) rot_prefetch(P.rot, 32 * warp, lane);
    // thread = dim; the rows' positions and elements, then their angles
    const RopeDim rd = rope_dim(P, t);
    const bool turned = t < P.rotary;
#pragma unroll 1
    for (int i0 = 0; i0 < kRows && r0 + i0 < total; i0 += 8) {
        float x[8], y[8], c[8], s[8];
        int pos[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t row = min(r0 + i0 + i, total - 1), n = div.div(row), h = row - n * H;
            pos[i] = position_of(P, (int)n);
            const T* p = base + (int64_t)n * sn + (int64_t)h * sh;
            x[i] = to_f32<T>(p[t]);
            y[i] = turned ? to_f32<T>(p[rd.partner]) : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float* cs = table_row<T>(P, pos[i]) + rd.j;
            c[i] = turned ? __ldg(cs) : 1.0f;
            s[i] = turned ? __ldg(cs + (P.rotary >> 1)) : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            // (rounded once; a query whose position is outside the table has
            // no value)
            float v = turned ? pair_rn(x[i], c[i], y[i], rd.sign * s[i]) : x[i];
            if (pos[i] < 0 && !keys) v = __int_as_float(0x7fc00000);
            xs[(i0 + i) * kPitch + t] = v;
        }
    }
    if constexpr (!k8) {
        if (t < nc - 1) smid[t] = __ldg(P.mids + t);
        if (t < nc) scent[t] = __ldg(P.cents + t);
    }
    __syncthreads();
    const int m = lane & 15, half = (lane >> 4) + 2 * warp;  // rows half and half + 8 of this half-warp
    float nsq[2] = {0.0f, 0.0f};
    if (keys && !k8) {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const float* x = xs + (half + 8 * k) * kPitch + 8 * m;
            float q = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) q = fmaf(x[j], x[j], q);
            nsq[k] = warp_sum_xor(q, 1, 8);
        }
    }
    if constexpr (!k8) {
        const int g = lane >> 2, c = lane & 3, n0 = 32 * warp;
        const float* R = P.rot + 4 * c * kHeadDim + n0 + 4 * g;
        const float* x = xs + g * kPitch + 4 * c;
        RotSums sums;
#pragma unroll 2
        for (int k = 0; k < kHeadDim; k += 16)
            rot_step<3, false>(sums, R, k, *reinterpret_cast<const float4*>(x + k),
                               *reinterpret_cast<const float4*>(x + 8 * kPitch + k));
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < 2; j++)
                *reinterpret_cast<float4*>(xs + (g + 8 * i) * kPitch + n0 + 8 * c + 4 * j) = sums.get(i, j);
        __syncthreads();
    }
    if (!keys) {
        for (int i = 0; i < kRows && r0 + i < total; i++) {
            const uint32_t n = div.div(r0 + i), h = (r0 + i) - n * H;
            P.q_rot[(int64_t)n * P.osn + (int64_t)h * P.osh + t] = xs[i * kPitch + t];
        }
        return;
    }
#pragma unroll 1
    for (int k = 0; k < 2; k++) {
        const uint32_t row = r0 + half + 8 * k;
        const bool live = row < total;
        const uint32_t rc = live ? row : total - 1;
        const uint32_t n = div.div(rc), h = rc - n * H;
        float z[8];
#pragma unroll
        for (int j = 0; j < 8; j++) z[j] = xs[(half + 8 * k) * kPitch + 8 * m + j];
        finish_row<T, L>(P, smid, scent, (int)n, (int)h, live, lane, z, k == 0 ? nsq[0] : nsq[1]);
    }
}

// ---------------------------------------------------------------------------
// Many rows of aligned inputs (Lloyd-Max layouts): the rotation on the tensor
// cores.  A persistent CTA walks tiles of 128 rows (of keys, then of queries):
//   warps 0-3    finish a tile: thread = row (= TMEM lane), its 128 coordinates
//                bucketised and packed, or written (queries);
//   warps 4-11   turn the next tile's rows and split them: x 2^s = hi + lo in
//                fp16 (22 bits), s from |x|; the first of them issues the
//                products;
//   warps 12-19  the values of the CTA's key rows, half a warp each.
// x R = hi R_hi + lo R_hi + hi R_lo in fp32 (R 2^10 split the same way, kept in
// shared memory): 24 MMAs of 128 x 128 x 16 a tile, the two small products
// first.  Errors against exact arithmetic, of |x|: 2^-23 from the fp32 turn, 3 *
// 2^-22 from the splits, 16 accumulations of 2^-23 at the size of the small
// products (2^-10) and 8 of 2^-23 at full size (kNear has the rest).
// Bound by instruction issue and latency: about 14 instructions per coordinate
// to bucketise, 9 to turn and split, 10 per value.  32768 tokens x 8 KV heads:
// 152 us (4, 6, 6 warps: 177; a second group of finishing warps changes
// nothing); 2037 tokens x 40 heads, 3-bit AoS: 35 us.
// ---------------------------------------------------------------------------
// Up to here the form above is faster: 5120 rows of a 4-bit decode step take it
// 15.8 us and this one 16.7, 10240 rows 21.5 and 17.5.
constexpr int64_t kFewRows = 6144;
constexpr int kATile = 128 * kHeadDim * 2;                                       // 32 KB
constexpr int kAHiOff = 0, kALoOff = kATile, kBHiOff = 2 * kATile, kBLoOff = 3 * kATile;
constexpr int kCells = 128;                                                      // of [-kCellSpan, kCellSpan)
constexpr float kCellSpan = 0.25f;
constexpr int kCellOff = 4 * kATile;                                             // [kCells][32 lanes]
constexpr int kTurnOff = kCellOff + kCells * 32 * 4;                             // 4 warps x 4 KB
constexpr int kInfoOff = kTurnOff + 4 * 4096;                                    // [2][128] RowInfo
constexpr int kRowOff = kInfoOff + 2 * 128 * 24;                                 // [128] element offsets of the rows
constexpr int kTabOff = kRowOff + 128 * 8;                                       // mids, c^2
constexpr int kUmmaBarOff = kTabOff + 2 * kNumCentroids * 4;
constexpr int kUmmaSmem = kUmmaBarOff + 64;
static_assert(kUmmaSmem <= 232448, "shared memory per CTA");
constexpr int kFinishWarps = 4, kTurnWarps = 8, kValueWarps = 8;
constexpr int kUmmaThreads = (kFinishWarps + kTurnWarps + kValueWarps) * 32;
enum : uint32_t { kAEmpty = 0, kDFull = 8, kDEmpty = 24, kUTmem = 40, kUAbort = 44 };

// What the finishing warps need of a row: the sum of squares, the factor that
// undoes the scales, its token, position and head, and its slot (-1: not
// stored; queries: -1 where the position is outside the table).
struct __align__(8) RowInfo {
    float nsq, unscale;
    int n, slot, pos, h;
};

template <typename T>
struct Quad {  // four consecutive elements, as loaded
    uint32_t w[sizeof(T)];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (sizeof(T) == 4) {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
            w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
        } else {
            const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
            w[0] = u.x; w[1] = u.y;
        }
    }
    __device__ __forceinline__ float operator[](int i) const {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(w[i]);
        } else {
            const unsigned short h = (unsigned short)(w[i >> 1] >> (16 * (i & 1)));
            return to_f32<T>(*reinterpret_cast<const T*>(&h));
        }
    }
};

struct UmmaTiles {
    uint32_t key_rows, rows, key_tiles, tiles;
};

// Row r of a tile: its token, head, slot and position.  (One row per thread, a
// tile ahead: these loads depend on one another.)
__device__ __forceinline__ RowInfo find_row(const AppendParams& P, const UmmaTiles& W, uint32_t tile, uint32_t r) {
    const bool keys = tile < W.key_tiles;
    const uint32_t total = keys ? W.key_rows : W.rows - W.key_rows, row = (keys ? tile : tile - W.key_tiles) * 128u + r;
    const FastDiv& div = keys ? P.div_hk : P.div_hq;
    const uint32_t at = min(row, total - 1), n = div.div(at);
    RowInfo x;
    x.n = (int)n;
    x.h = (int)(at - n * (uint32_t)(keys ? P.Hk : P.Hq));
    x.pos = position_of(P, (int)n);
    x.slot = row >= total ? -1 : keys ? __ldg(P.slots + n) : 0;
    if (keys && P.num_blocks > 0 && (int64_t)x.slot >= P.num_blocks * kBlockSize) x.slot = -1;
    x.slot = x.pos < 0 ? -1 : max(x.slot, -1);
    x.nsq = x.unscale = 0.0f;
    return x;
}

// A tile's rows turned, scaled, split and stored (128-byte swizzle, K-major),
// half a warp per row: lane m of 16 takes pairs 4m .. 4m + 3 of the row's 64
// (pairs that the rotary step turns together, and the rest two by two).
template <typename T>
__device__ __forceinline__ void turn_rows(const AppendParams& P, uint8_t* smem, bool keys, int buf, int lw, int lane) {
    const T* base = static_cast<const T*>(keys ? P.key : P.query);
    RowInfo* infos = reinterpret_cast<RowInfo*>(smem + kInfoOff) + 128 * buf;
    const int64_t* offs = reinterpret_cast<const int64_t*>(smem + kRowOff);
    const int m = lane & 15, half = P.rotary >> 1, j0 = 4 * m;
    const bool turned = j0 < half;
    // dims of the lane's pairs: (a, b) = (da + i, db + i), or interleaved
    // (2 j, 2 j + 1)
    int da, db;
    if (P.interleaved) {
        da = 2 * j0;
        db = da + 4;
    } else {
        da = turned ? j0 : P.rotary + (j0 - half);
        db = turned ? j0 + half : P.rotary + (64 - half) + (j0 - half);
    }
    // One piece of code for both rotary rules (four roles run at once, and their
    // instructions have to stay in the caches), two rows at a time; the next
    // two are loaded while these are turned.
    struct Row {
        Quad<T> a, b;
        float4 c, s;
    };
    constexpr int kBatch = 2, kStep = 2 * kTurnWarps;  // rows of the role's warps together
    Row x0[kBatch], x1[kBatch];
    const int hw = lane >> 4, r_first = 2 * lw + hw;
    auto load = [&](Row (&x)[kBatch], int r0) {
#pragma unroll
        for (int i = 0; i < kBatch; i++) {
            const int r = min(r0 + kStep * i, 127);
            const T* p = base + offs[r];
            x[i].a.load(p + da);
            x[i].b.load(p + db);
            x[i].c = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
            x[i].s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (turned) {
                const float* cs = table_row<T>(P, infos[r].pos) + j0;
                x[i].c = __ldg(reinterpret_cast<const float4*>(cs));
                x[i].s = __ldg(reinterpret_cast<const float4*>(cs + half));
            }
        }
    };
    auto turn = [&](const Row (&now)[kBatch], int r0) {
#pragma unroll
        for (int i = 0; i < kBatch; i++) {
            const int r = r0 + kStep * i;
            if (r - hw >= 128) break;  // (the warp's halves stay together)
            const float cc[4] = {now[i].c.x, now[i].c.y, now[i].c.z, now[i].c.w};
            const float ss[4] = {now[i].s.x, now[i].s.y, now[i].s.z, now[i].s.w};
            const float in[8] = {now[i].a[0], now[i].a[1], now[i].a[2], now[i].a[3],
                                 now[i].b[0], now[i].b[1], now[i].b[2], now[i].b[3]};
            float u[4], v[4], x[8];  // the pairs, then dims da .. da + 3, db .. db + 3
            float nsq = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float ak = P.interleaved ? in[2 * k] : in[k], bk = P.interleaved ? in[2 * k + 1] : in[4 + k];
                u[k] = fmaf(ak, cc[k], -(bk * ss[k]));
                v[k] = fmaf(bk, cc[k], ak * ss[k]);
                nsq = fmaf(u[k], u[k], fmaf(v[k], v[k], nsq));
            }
            nsq = warp_sum_xor(nsq, 1, 8);
            // |x| 2^e in [2^13, 2^15): e from the exponent of |x|^2 (its half,
            // rounded up); 0 where |x|^2 is 0 or not finite (keys: the exact path
            // or no codes; queries: exact_queries)
            const int be = (int)(__float_as_uint(nsq) >> 23);
            const int e = be == 0 || be == 0xFF ? 0 : 14 - ((be - 126) >> 1);
            const float f = exp2i(e);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                x[k] = (P.interleaved ? (k & 1 ? v[k >> 1] : u[k >> 1]) : u[k]) * f;
                x[4 + k] = (P.interleaved ? (k & 1 ? v[2 + (k >> 1)] : u[2 + (k >> 1)]) : v[k]) * f;
            }
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const __half2 h = __floats2half2_rn(x[2 * k], x[2 * k + 1]);
                hi[k] = h2_as_u32(h);
                lo[k] = h2_as_u32(__floats2half2_rn(x[2 * k] - __low2float(h), x[2 * k + 1] - __high2float(h)));
            }
            // four dims are 8 bytes of a 16-byte chunk
            auto at = [&](int d) { return (d >> 6) * (kATile / 2) + r * 128 + ((((d & 63) >> 3) ^ (r & 7)) << 4) + (d & 4) * 2; };
            *reinterpret_cast<uint2*>(smem + kAHiOff + at(da)) = make_uint2(hi[0], hi[1]);
            *reinterpret_cast<uint2*>(smem + kAHiOff + at(db)) = make_uint2(hi[2], hi[3]);
            *reinterpret_cast<uint2*>(smem + kALoOff + at(da)) = make_uint2(lo[0], lo[1]);
            *reinterpret_cast<uint2*>(smem + kALoOff + at(db)) = make_uint2(lo[2], lo[3]);
            if (m == 0) *reinterpret_cast<float2*>(infos + r) = make_float2(nsq, exp2i(-e) * 0x1p-10f);
        }
    };
    // (two buffers by name: handing one's registers to the other would wait for
    // its loads)
    constexpr int kNext = kStep * kBatch;
    load(x0, r_first);
#pragma unroll 1
    for (int r0 = r_first; r0 - hw < 128; r0 += 2 * kNext) {
        load(x1, r0 + kNext);
        turn(x0, r0);
        load(x0, r0 + 2 * kNext);
        turn(x1, r0 + kNext);
    }
}

// Asks L2 for a tile's rows (thread t of `threads`).
template <typename T>
__device__ __forceinline__ void prefetch_rows(const T* base, int64_t sn, int64_t sh, const FastDiv& div, uint32_t H, uint32_t first,
                                              uint32_t total, int t, int threads) {
    constexpr int kLines = sizeof(T);  // 128-byte lines of a row
    for (uint32_t line = (uint32_t)t; line < 128u * kLines; line += (uint32_t)threads) {
        const uint32_t row = first + line / kLines;
        if (row < total) {
            const uint32_t n = div.div(row), h = row - n * H;
            asm volatile("prefetch.global.L2 [%0];\n" ::"l"(base + (int64_t)n * sn + (int64_t)h * sh + (line % kLines) * (128 / kLines)));
        }
    }
}

// A row's elements: all zero (a sum of squares of 0 may also be that of small
// numbers), all finite, or not.
enum Elements : int { kZeros, kFinite, kNonFinite };
template <typename T>
__device__ __noinline__ Elements elements(const T* row) {
    bool some = false, finite = true;
#pragma unroll 4
    for (int d = 0; d < kHeadDim; d += 4) {
        Quad<T> x;
        x.load(row + d);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            some |= x[i] != 0.0f;
            finite &= isfinite(x[i]);
        }
    }
    return !some ? kZeros : finite ? kFinite : kNonFinite;
}
// The codes of a row of zeros.
template <int L>
__device__ __noinline__ void zero_codes(uint8_t* key, const float* smid) {
    constexpr bool k3 = layout_3bit_keys(L);
    uint32_t code = 0;
    for (int k = 0; k < (k3 ? 8 : kNumCentroids) - 1; k++) code += smid[k] <= 0.0f ? 1u : 0u;
    const uint64_t codes = code * (k3 ? 0x249249249249ull : 0x1111111111111111ull);
    for (int i = 0; i < aos_key_bytes(L) / 2; i++)
        reinterpret_cast<unsigned short*>(key)[i] = (unsigned short)(codes >> (16 * (i % (k3 ? 3 : 4))));
}

// A key row: codes of its 128 coordinates, norm, slot.
template <typename T, int L>
__device__ __forceinline__ void finish_keys(const AppendParams& P, uint8_t* smem, uint32_t tm, const RowInfo& info,
                                            bool fine, int lane) {
    constexpr bool k3 = layout_3bit_keys(L);
    constexpr int nc = k3 ? 8 : kNumCentroids, kBits = k3 ? 3 : 4;
    constexpr unsigned kFull = 0xffffffffu;
    const float* smid = reinterpret_cast<const float*>(smem + kTabOff);
    const float* csq16 = smid + kNumCentroids;
    const float norm = __fsqrt_rn(info.nsq);
    const float f = info.unscale * __frcp_rn(norm + 1e-8f);
    const uint32_t h = (uint32_t)info.h;
    const uint8_t* cells = smem + kCellOff + 4 * lane;
    const bool stored = info.slot >= 0;
    const uint32_t slot = stored ? (uint32_t)info.slot : 0u;
    const SlotAt<L> at(P.cache + (size_t)(slot / kBlockSize) * (size_t)P.block_bytes, slot % kBlockSize, h, P.Hk, P.pos_stride,
                       P.head_stride);
    // A row of zeros (dummy inputs): every coordinate is 0 exactly, and next to
    // a middle border all 128 would go through 64 bits (4096 tokens x 8 heads:
    // 5.8 ms, 25 us for random ones).  Its codes are written again below.
    const bool zeros = stored && info.nsq == 0.0f &&
                       elements<T>(static_cast<const T*>(P.key) + (int64_t)info.n * P.ksn + (int64_t)info.h * P.ksh) == kZeros;
    float csq = 0.0f;
#pragma unroll 1
    for (int q = 0; q < 8; q++) {
        float part = 0.0f;  // of csq: one chain of 128 additions would be off by 2^-17
        uint32_t z[16];
        tmem_ld16(z, tm + 16 * q);
        tmem_wait_ld();
        uint32_t near = 0u;   // coordinates next to a border
        uint64_t codes = 0u;  // 16 of them
        if (fine) {
#pragma unroll
            for (int j = 0; j < 16; j++) {
                const float y = __uint_as_float(z[j]) * f;
                // the nearest border of y's cell, its index in the low bits
                // (t counts 128ths of cells, so that its integer is the byte offset)
                const float t = fminf(fmaxf(fmaf(y, 128.0f * kCells / (2.0f * kCellSpan), 0x1p23f + 64.0f * kCells + 64.0f), 0x1p23f),
                                      0x1p23f + (128.0f * kCells - 1.0f));
                const uint32_t e = *reinterpret_cast<const uint32_t*>(cells + (__float_as_uint(t) & (128u * (kCells - 1))));
                const float d = y - __uint_as_float(e);
                const int code = (int)(e & 15u) + (d >= 0.0f ? 1 : 0);
                part += csq16[code];
                near |= fabsf(d) < kNear ? 1u << j : 0u;
                codes |= (uint64_t)(uint32_t)code << (kBits * j);
            }
        } else {  // by search
#pragma unroll 1
            for (int j = 0; j < 16; j++) {
                float y = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; i++) y = i == j ? __uint_as_float(z[i]) * f : y;
                int code = 0;
                for (int k = 0; k < nc - 1; k++) code += y >= smid[k] ? 1 : 0;
                part += csq16[code];
                near |= (code > 0 && y - smid[max(code - 1, 0)] < kNear) || (code < nc - 1 && smid[code] - y < kNear) ? 1u << j : 0u;
                codes |= (uint64_t)(uint32_t)code << (kBits * j);
            }
        }
        // in 64 bits by the whole warp (a row that is not stored needs none)
        if (!stored || zeros) near = 0u;
        uint32_t who;
        while ((who = __ballot_sync(kFull, near != 0u)) != 0u) {
            const int src = __ffs(who) - 1;
            const int sn = __shfl_sync(kFull, info.n, src), sh = __shfl_sync(kFull, (int)h, src);
            const int j = __shfl_sync(kFull, __ffs(near) - 1, src);
            const T* krow = static_cast<const T*>(P.key) + (int64_t)sn * P.ksn + (int64_t)sh * P.ksh;
            const int c = exact_code<T>(P, krow, table_row<T>(P, __shfl_sync(kFull, info.pos, src)), 16 * q + j, smid, nc - 1, lane);
            if (lane == src) {
                const int c0 = (int)(codes >> (kBits * j)) & (nc - 1);
                near &= near - 1;
                part += csq16[c] - csq16[c0];
                codes ^= (uint64_t)(uint32_t)(c ^ c0) << (kBits * j);
            }
        }
        csq += part;
        if (stored) {
            if constexpr (k3) {
#pragma unroll
                for (int i = 0; i < 3; i++)
                    reinterpret_cast<unsigned short*>(at.key)[3 * q + i] = (unsigned short)(codes >> (16 * i));
            } else if constexpr (layout_is_aos(L)) {
                st_u16x2(at.key + 8 * q, (uint32_t)codes);
                st_u16x2(at.key + 8 * q + 4, (uint32_t)(codes >> 32));
            } else {
                reinterpret_cast<uint2*>(at.key)[q] = make_uint2((uint32_t)codes, (uint32_t)(codes >> 32));
            }
        }
    }
    if (zeros) zero_codes<L>(at.key, smid);
    const bool fold = !layout_is_aos(L) && P.norm_correction;
    const float kept = fold ? norm * rsqrtf(csq + 1e-16f) : norm;
    unsigned short kept_h = __half_as_ushort(__float2half_rn(kept));
    // (NaN too: turn_rows makes it of infinite elements that it does not turn)
    const bool split = stored && !__heq(__float2half_rn(kept * (1.0f - kNormNear)), __float2half_rn(kept * (1.0f + kNormNear)));
    uint32_t ask = __ballot_sync(kFull, split);
    while (ask != 0u) {
        const int src = __ffs(ask) - 1;
        ask &= ask - 1;
        const int sn = __shfl_sync(kFull, info.n, src), sh = __shfl_sync(kFull, (int)h, src);
        const T* krow = static_cast<const T*>(P.key) + (int64_t)sn * P.ksn + (int64_t)sh * P.ksh;
        double v = exact_norm<T>(P, krow, table_row<T>(P, __shfl_sync(kFull, info.pos, src)), lane);
        if (fold) {
            // the codes just written: four per lane, from the row's bytes
            __syncwarp();
            const uint8_t* codes = reinterpret_cast<const uint8_t*>(__shfl_sync(kFull, reinterpret_cast<unsigned long long>(at.key), src));
            double cq = 0.0;
            for (int i = 0; i < 4; i++) {
                const int bit = kBits * (4 * lane + i);
                const volatile uint8_t* b = codes + (bit >> 3);
                const uint32_t two = (uint32_t)b[0] | ((bit & 7) + kBits > 8 ? (uint32_t)b[1] << 8 : 0u);
                const double cv = (double)__ldg(P.cents + ((two >> (bit & 7)) & (nc - 1)));
                cq += cv * cv;
            }
            v /= sqrt(warp_sum_f64(cq) + 1e-16);
        }
        // (one NaN for both forms: the float conversion's)
        if (lane == src) kept_h = __half_as_ushort(v != v ? __float2half_rn((float)v) : __double2half(v));
    }
    if (stored) *reinterpret_cast<unsigned short*>(at.norm) = kept_h;
}

// The lanes' query rows (token n, head h) that are `odd`, in 64 bits (whole
// warp); rows of zeros and rows that are not finite are left as they are.
template <typename T>
__device__ __noinline__ void exact_queries(const AppendParams& P, int n, int h, int pos, bool odd, int lane) {
    constexpr unsigned kFull = 0xffffffffu;
    uint32_t who = __ballot_sync(
        kFull, odd && elements<T>(static_cast<const T*>(P.query) + (int64_t)n * P.qsn + (int64_t)h * P.qsh) == kFinite);
    while (who != 0u) {
        const int src = __ffs(who) - 1;
        who &= who - 1;
        const int64_t sn = __shfl_sync(kFull, n, src), sh = __shfl_sync(kFull, h, src);
        const T* row = static_cast<const T*>(P.query) + sn * P.qsn + sh * P.qsh;
        const float* cs = table_row<T>(P, __shfl_sync(kFull, pos, src));
        double z[4] = {};
#pragma unroll 1
        for (int d = 0; d < kHeadDim; d++) {
            const double x = rope_f64<T>(P, row, cs, d);
            const float4 r = __ldg(reinterpret_cast<const float4*>(P.rot + d * kHeadDim) + lane);
            z[0] += x * (double)r.x;
            z[1] += x * (double)r.y;
            z[2] += x * (double)r.z;
            z[3] += x * (double)r.w;
        }
        reinterpret_cast<float4*>(P.q_rot + sn * P.osn + sh * P.osh)[lane] =
            make_float4((float)z[0], (float)z[1], (float)z[2], (float)z[3]);
    }
}

// Query rows: the product itself, turned through shared memory into runs of
// 128 bytes.
template <typename T>
__device__ __forceinline__ void finish_queries(const AppendParams& P, uint8_t* turn, uint32_t tm,
                                               const RowInfo& info, bool live, int lane) {
    float* dst = P.q_rot + (int64_t)info.n * P.osn + (int64_t)info.h * P.osh;
    const float f = info.slot < 0 ? __int_as_float(0x7fc00000) : info.unscale;
    const uint32_t live_rows = __ballot_sync(0xffffffffu, live);
    const unsigned long long mine = reinterpret_cast<unsigned long long>(dst);
    float* rows[8];
#pragma unroll
    for (int i = 0; i < 8; i++)
        rows[i] = reinterpret_cast<float*>(__shfl_sync(0xffffffffu, mine, 4 * i + (lane >> 3))) + 4 * (lane & 7);
#pragma unroll 1
    for (int q = 0; q < 4; q++) {
        uint32_t z[32];
        tmem_ld32(z, tm + 32 * q);
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < 8; c++)
            *reinterpret_cast<float4*>(turn + 128 * lane + ((c ^ (lane & 7)) << 4)) =
                make_float4(__uint_as_float(z[4 * c]) * f, __uint_as_float(z[4 * c + 1]) * f,
                            __uint_as_float(z[4 * c + 2]) * f, __uint_as_float(z[4 * c + 3]) * f);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int r = 4 * i + (lane >> 3);
            const float4 v = *reinterpret_cast<const float4*>(turn + 128 * r + (((lane & 7) ^ (r & 7)) << 4));
            if ((live_rows >> r) & 1u) *reinterpret_cast<float4*>(rows[i] + 32 * q) = v;
        }
        __syncwarp();
    }
    // rows whose squares leave fp32's range, and with them the split's scale
    const bool odd = live && info.slot >= 0 && (info.nsq < 0x1p-120f || info.nsq == INFINITY);
    if (__any_sync(0xffffffffu, odd)) exact_queries<T>(P, info.n, info.h, info.pos, odd, lane);
}

// The values of a tile's rows, half a warp each, two at a time with the next
// two in flight.
template <typename T, int L>
__device__ __forceinline__ void store_values(const AppendParams& P, const UmmaTiles& W, uint32_t tile, int vw, int lane) {
    const int m = lane & 15;
    constexpr int kBatch = 2, kStep = 2 * kValueWarps;
    struct Row {
        Quad<T> a, b;
        int slot, pos;
        uint32_t h;
    };
    Row x0[kBatch], x1[kBatch];
    auto load = [&](Row (&x)[kBatch], int r0) {
#pragma unroll
        for (int i = 0; i < kBatch; i++) {
            const int r = r0 + kStep * i;
            const uint32_t row0 = tile * 128u + r, row = min(row0, W.key_rows - 1);
            const uint32_t n = P.div_hk.div(row);
            x[i].h = row - n * (uint32_t)P.Hk;
            const T* v = static_cast<const T*>(P.value) + (int64_t)n * P.vsn + (int64_t)x[i].h * P.vsh + 8 * m;
            x[i].a.load(v);
            x[i].b.load(v + 4);
            x[i].slot = r < 128 && row0 < W.key_rows ? __ldg(P.slots + n) : -1;
            x[i].pos = position_of(P, (int)n);
        }
    };
    auto store = [&](const Row (&x)[kBatch], int r0) {
#pragma unroll
        for (int i = 0; i < kBatch; i++) {
            if (r0 + kStep * i - (lane >> 4) >= 128) break;  // (the warp's halves stay together)
            const float v[8] = {x[i].a[0], x[i].a[1], x[i].a[2], x[i].a[3], x[i].b[0], x[i].b[1], x[i].b[2], x[i].b[3]};
            const ValueRow q = quantise_values<layout_3bit_values(L)>(v);
            const int slot = x[i].slot;
            if (slot >= 0 && x[i].pos >= 0 && (P.num_blocks <= 0 || (int64_t)slot < P.num_blocks * kBlockSize))
                write_values<L>(SlotAt<L>(P.cache + (size_t)((uint32_t)slot / kBlockSize) * (size_t)P.block_bytes,
                                          (uint32_t)slot % kBlockSize, x[i].h, P.Hk, P.pos_stride, P.head_stride),
                                m, q);
        }
    };
    constexpr int kNext = kStep * kBatch;
    const int r_first = 2 * vw + (lane >> 4);
    load(x0, r_first);
#pragma unroll 1
    for (int r0 = r_first; r0 - (lane >> 4) < 128; r0 += 2 * kNext) {
        load(x1, r0 + kNext);
        store(x0, r0);
        load(x0, r0 + 2 * kNext);
        store(x1, r0 + kNext);
    }
}

template <typename T, int L>
__global__ void __launch_bounds__(kUmmaThreads, 1) append_umma_kernel(const __grid_constant__ AppendParams P,
                                                                      const UmmaTiles W) {
    constexpr bool k3 = layout_3bit_keys(L);
    constexpr int nc = k3 ? 8 : kNumCentroids;
    extern __shared__ __align__(1024) uint8_t smem[];
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const uint32_t base = smem_addr(smem), bars = base + kUmmaBarOff;
    volatile uint32_t* abort = reinterpret_cast<volatile uint32_t*>(smem + kUmmaBarOff + kUAbort);
    if (tid == 0) {
        bar_init(bars + kAEmpty, 1);
        for (int b = 0; b < 2; b++) {
            bar_init(bars + kDFull + 8 * b, 1);
            bar_init(bars + kDEmpty + 8 * b, 128);
        }
        *abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == kFinishWarps) tmem_alloc<256>(bars + kUTmem);
    float* smid = reinterpret_cast<float*>(smem + kTabOff);
    if (tid < kNumCentroids) {
        smid[tid] = tid < nc - 1 ? __ldg(P.mids + tid) : INFINITY;
        const float c = tid < nc ? __ldg(P.cents + tid) : 0.0f;
        smid[kNumCentroids + tid] = c * c;
    }
    // R 2^10 = hi + lo, [64 columns][128 rows of 128 bytes], swizzled: the
    // MN-major B operand
    for (int i = tid; i < kHeadDim * kHeadDim / 8; i += kUmmaThreads) {
        const int d = i >> 4, c = i & 15;  // row, group of 8 columns
        const float4 u = __ldg(reinterpret_cast<const float4*>(P.rot + d * kHeadDim + 8 * c));
        const float4 v = __ldg(reinterpret_cast<const float4*>(P.rot + d * kHeadDim + 8 * c + 4));
        const float x[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float a = x[2 * k] * 1024.0f, b = x[2 * k + 1] * 1024.0f;
            const __half2 h = __floats2half2_rn(a, b);
            hi[k] = h2_as_u32(h);
            lo[k] = h2_as_u32(__floats2half2_rn(a - __low2float(h), b - __high2float(h)));
        }
        const int at = (c >> 3) * (kATile / 2) + d * 128 + (((c & 7) ^ (d & 7)) << 4);
        *reinterpret_cast<uint4*>(smem + kBHiOff + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(smem + kBLoOff + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
    fence_async_smem();
    __syncthreads();
    // Cells of the coordinate's range: the border nearest to the cell, its
    // index in the four low bits (at most 15 units of 2^-26, see kNear).  A cell
    // that two borders come near to leaves every row to the search.
    bool fine = true;
    if (tid < kCells) {
        const float w = 2.0f * kCellSpan / kCells, mid = -kCellSpan + w * ((float)tid + 0.0f);
        // cells are centred on mid (the index is rounded); the outer two reach on
        int best = 0, inside = 0;
        for (int k = 0; k < nc - 1; k++) {
            if (fabsf(smid[k] - mid) < fabsf(smid[best] - mid)) best = k;
            if (fabsf(smid[k] - mid) < 0.75f * w) inside++;
        }
        fine = inside <= 1 && smid[0] > -kCellSpan + w && smid[nc - 2] < kCellSpan - 2.0f * w;
        uint32_t* cell = reinterpret_cast<uint32_t*>(smem + kCellOff) + 32 * tid;
        const uint32_t e = (__float_as_uint(smid[best]) & ~15u) | (uint32_t)best;
        for (int i = 0; i < 32; i++) cell[(i + lane) & 31] = e;
    }
    fine = __syncthreads_and(fine) != 0;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + kUmmaBarOff + kUTmem);

    if (warp < kFinishWarps) {
        const int wq = warp;
        uint32_t i = 0;
        for (uint32_t tile = blockIdx.x; tile < W.tiles; tile += gridDim.x, i++) {
            const int g = (int)(i & 1);
            if (!bar_wait_warp(bars + kDFull + 8 * g, (i >> 1) & 1, abort)) break;
            tc_fence_after();
            const bool keys = tile < W.key_tiles;
            const uint32_t row = (keys ? tile : tile - W.key_tiles) * 128u + 32u * wq + lane;
            const bool live = row < (keys ? W.key_rows : W.rows - W.key_rows);
            const RowInfo info = reinterpret_cast<const RowInfo*>(smem + kInfoOff)[g * 128 + 32 * wq + lane];
            const uint32_t tm = tmem + ((uint32_t)(32 * wq) << 16) + 128u * g;
            if (__any_sync(0xffffffffu, live)) {
                if (keys)
                    finish_keys<T, L>(P, smem, tm, info, fine, lane);
                else
                    finish_queries<T>(P, smem + kTurnOff + 4096 * warp, tm, info, live, lane);
            }
            tc_fence_before();
            bar_arrive(bars + kDEmpty + 8 * g);
        }
    } else if (warp < kFinishWarps + kTurnWarps) {
        constexpr uint32_t kId = umma_idesc(128, kHeadDim, true);
        const uint64_t a_hi = umma_desc(base + kAHiOff, 16, 1024), a_lo = umma_desc(base + kALoOff, 16, 1024);
        const uint64_t b_hi = umma_desc(base + kBHiOff, kATile / 2, 1024), b_lo = umma_desc(base + kBLoOff, kATile / 2, 1024);
        uint32_t i = 0;
        bool ok = true;
        const int t = tid - 32 * kFinishWarps;
        RowInfo mine{};  // row t of the next tile
        if (t < 128 && blockIdx.x < W.tiles) mine = find_row(P, W, blockIdx.x, (uint32_t)t);
        for (uint32_t tile = blockIdx.x; tile < W.tiles; tile += gridDim.x, i++) {
            const int buf = (int)(i & 1);
            // the operands' last readers, and the rows' (their infos and sums)
            ok = ok && bar_wait_warp(bars + kAEmpty, (i & 1) ^ 1, abort) &&
                 bar_wait_warp(bars + kDEmpty + 8 * buf, ((i >> 1) & 1) ^ 1, abort);
            const uint32_t next = tile + gridDim.x;
            if (next < W.key_tiles)
                prefetch_rows<T>(static_cast<const T*>(P.key), P.ksn, P.ksh, P.div_hk, (uint32_t)P.Hk, next * 128u, W.key_rows,
                                 t, 32 * kTurnWarps);
            else if (next < W.tiles)
                prefetch_rows<T>(static_cast<const T*>(P.query), P.qsn, P.qsh, P.div_hq, (uint32_t)P.Hq,
                                 (next - W.key_tiles) * 128u, W.rows - W.key_rows,
                                 t, 32 * kTurnWarps);
            const bool keys = tile < W.key_tiles;
            if (ok && t < 128) {
                reinterpret_cast<RowInfo*>(smem + kInfoOff)[128 * buf + t] = mine;
                reinterpret_cast<int64_t*>(smem + kRowOff)[t] =
                    (int64_t)mine.n * (keys ? P.ksn : P.qsn) + (int64_t)mine.h * (keys ? P.ksh : P.qsh);
            }
            asm volatile("bar.sync 2, %0;\n" ::"n"(32 * kTurnWarps) : "memory");
            if (t < 128 && next < W.tiles) mine = find_row(P, W, next, (uint32_t)t);
            if (ok) turn_rows<T>(P, smem, keys, buf, warp - kFinishWarps, lane);
            fence_async_smem();
            asm volatile("bar.sync 1, %0;\n" ::"n"(32 * kTurnWarps) : "memory");  // every warp takes every turn, also after an error
            if (ok && warp == kFinishWarps) {
                tc_fence_after();
#pragma unroll
                for (int p = 0; p < 3; p++)
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        const uint64_t at = ((k >> 2) * (kATile / 2) + (k & 3) * 32) >> 4;
                        umma_ss(tmem + 128u * buf, (p == 0 ? a_lo : a_hi) + at, (p == 1 ? b_lo : b_hi) + (k * 2048 >> 4), kId,
                                p + k != 0);
                    }
                umma_commit(bars + kDFull + 8 * buf);
                umma_commit(bars + kAEmpty);
            }
        }
        // every product has ended before the CTA frees its TMEM
        if (warp == kFinishWarps && i > 0) bar_wait_warp(bars + kAEmpty, (i - 1) & 1, nullptr);
    } else {
        for (uint32_t tile = blockIdx.x; tile < W.key_tiles; tile += gridDim.x) {
            prefetch_rows<T>(static_cast<const T*>(P.value), P.vsn, P.vsh, P.div_hk, (uint32_t)P.Hk, (tile + gridDim.x) * 128u,
                             W.key_rows, tid - 32 * (kFinishWarps + kTurnWarps), 32 * kValueWarps);
            store_values<T, L>(P, W, tile, warp - kFinishWarps - kTurnWarps, lane);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kFinishWarps) tmem_free<256>(tmem);
    if (tid == 0 && *abort != 0) atomicAdd(&g_append_timeouts, 1u);
}

// Inputs that the tensor-core form reads with 8- and 16-byte loads: elements in
// fours, rotary halves in fours, SoA slots in 16 bytes.
template <typename T, int L>
bool umma_aligned(const AppendParams& P) {
    const uintptr_t a = 4 * sizeof(T);
    auto ok = [&](const void* p, int64_t sn, int64_t sh) {
        return reinterpret_cast<uintptr_t>(p) % a == 0 && sn % 4 == 0 && sh % 4 == 0;
    };
    return ok(P.key, P.ksn, P.ksh) && ok(P.value, P.vsn, P.vsh) && (!P.query || ok(P.query, P.qsn, P.qsh)) &&
           (!P.query || (reinterpret_cast<uintptr_t>(P.q_rot) % 16 == 0 && P.osn % 4 == 0 && P.osh % 4 == 0)) &&
           P.rotary % 8 == 0 && (!P.pos || (reinterpret_cast<uintptr_t>(P.cos_sin) % 16 == 0 && P.cs_stride % 4 == 0)) &&
           (layout_is_aos(L) || (reinterpret_cast<uintptr_t>(P.cache) % 16 == 0 && P.block_bytes % 16 == 0));
}

template <typename T, int L>
int launch_append_umma(const AppendParams& P, cudaStream_t stream, int num_sms) {
    auto kern = append_umma_kernel<T, L>;
    static thread_local int configured_dev = -1;
    int dev = 0;
    cudaGetDevice(&dev);
    if (configured_dev != dev) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kUmmaSmem) != cudaSuccess)
            return report_launch(cudaGetLastError());
        configured_dev = dev;
    }
    UmmaTiles W;
    W.key_rows = (uint32_t)P.N * (uint32_t)P.Hk;
    const uint32_t q_rows = P.query ? (uint32_t)P.N * (uint32_t)P.Hq : 0u;
    W.rows = W.key_rows + q_rows;
    W.key_tiles = (W.key_rows + 127) / 128;
    W.tiles = W.key_tiles + (q_rows + 127) / 128;
    const unsigned grid = W.tiles < (uint32_t)num_sms ? W.tiles : (unsigned)num_sms;
    kern<<<grid, kUmmaThreads, kUmmaSmem, stream>>>(P, W);
    return report_launch(cudaGetLastError());
}

template <typename T, int L>
int launch_append_t(const AppendParams& P, cudaStream_t stream, int num_sms) {
    const int64_t kr = (int64_t)P.N * P.Hk, qr = P.query ? (int64_t)P.N * P.Hq : 0;
    if constexpr (!layout_fp8_keys(L))
        if (kr + qr > kFewRows && umma_aligned<T, L>(P)) return launch_append_umma<T, L>(P, stream, num_sms);
    const int64_t kc = (kr + kRows - 1) / kRows, qc = (qr + kRows - 1) / kRows;
    append_kernel<T, L><<<(unsigned)(kc + qc), kAppThreads, 0, stream>>>(P, (int)kc);
    return report_launch(cudaGetLastError());
}

template <typename T>
int launch_append_d(const AppendParams& P, cudaStream_t stream, int num_sms) {
    switch (P.layout) {
        case TQB_LAYOUT_SOA: return launch_append_t<T, TQB_LAYOUT_SOA>(P, stream, num_sms);
        case TQB_LAYOUT_SOA_K8: return launch_append_t<T, TQB_LAYOUT_SOA_K8>(P, stream, num_sms);
        case TQB_LAYOUT_SOA_K3: return launch_append_t<T, TQB_LAYOUT_SOA_K3>(P, stream, num_sms);
        case TQB_LAYOUT_SOA_K3V3: return launch_append_t<T, TQB_LAYOUT_SOA_K3V3>(P, stream, num_sms);
        case TQB_LAYOUT_AOS: return launch_append_t<T, TQB_LAYOUT_AOS>(P, stream, num_sms);
        case TQB_LAYOUT_AOS_K8: return launch_append_t<T, TQB_LAYOUT_AOS_K8>(P, stream, num_sms);
        case TQB_LAYOUT_AOS_K3: return launch_append_t<T, TQB_LAYOUT_AOS_K3>(P, stream, num_sms);
        case TQB_LAYOUT_AOS_K3V3: return launch_append_t<T, TQB_LAYOUT_AOS_K3V3>(P, stream, num_sms);
        default: return TQB_ERR_INVALID_ARG;
    }
}

}  // namespace

int launch_append(const AppendParams& P, cudaStream_t stream, int num_sms) {
    if (P.N == 0) return TQB_OK;
    switch (P.dtype) {
        case TQB_DTYPE_F32: return launch_append_d<float>(P, stream, num_sms);
        case TQB_DTYPE_F16: return launch_append_d<__half>(P, stream, num_sms);
        case TQB_DTYPE_BF16: return launch_append_d<__nv_bfloat16>(P, stream, num_sms);
        default: return TQB_ERR_INVALID_ARG;
    }
}

int read_append_timeouts(unsigned int* count, bool reset) {
    cudaError_t e = cudaMemcpyFromSymbol(count, g_append_timeouts, sizeof(unsigned int));
    if (e == cudaSuccess && reset) {
        const unsigned int zero = 0;
        e = cudaMemcpyToSymbol(g_append_timeouts, &zero, sizeof(unsigned int));
    }
    return e == cudaSuccess ? TQB_OK : report_launch(e);
}

}  // namespace tqb
