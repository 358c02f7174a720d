// tqb_prefix.cu — decode attention over a prefix that every sequence of the
// batch shares, computed once for all of them on the 5th-generation tensor
// cores.
//
// For KV head h the rows are the queries of its G heads in all B sequences
// (R = B G of them), and for a chunk of the prefix's tokens T
//     S = Q K^T,  P = exp2(S kfac - m),  l = sum P,  O = P V / l,
// the softmax-normalised partial output and natural-log LSE of the chunk, in
// Stage1's mid_o form; Stage2 merges the chunks with each sequence's own
// tokens.  Per-sequence Stage1 dequantises the prefix B times; here a CTA
// dequantises a 128-token tile once for up to 256 rows.
//
// One CTA per SM, one (chunk, KV head, block of 256 rows); warps:
//   0-3, 4-7   streams 0 and 1: thread = row (= TMEM lane).  A stream is 128
//              rows over every tile, or with at most 128 rows the same rows
//              over the even or the odd tiles, so that two tiles are always in
//              flight.  Its four warps weigh a tile's scores, then its first
//              warp issues the products of these weights and the next tile's
//              scores;
//   8-11       dequantise K and V tiles (fp16, 128-byte swizzle) into two
//              stages of shared memory, the next tile's codes in registers.
// S = Q K^T has its operands in shared memory; P overwrites S in TMEM and is
// the A operand of O += P V there.  One stream's MMAs run under the other's
// softmax.  TMEM: S0 S1 O0 O1 of 128 columns each, all 512, so there is one S
// per stream.  (Measured at 256 rows x 32768 tokens x 8 heads, us: 57 with
// warps of their own that issue, whose waits and commits cost 130 and 200
// cycles each on the way from P to S; 52 with half tiles and two S per stream,
// a 128 x 64 x 16 product taking the tensor core as long as 128 x 128 x 16.)
//
// Precision: Q (scaled per row by a power of two), K = c norm, V = code scale
// + zero and P are rounded to fp16, each product accumulated in fp32; m, l, O
// and the LSE are fp32.  V's and P's errors average out over the tokens.  A
// score's (q, c and c norm rounded) grows with the scores, and a codebook's few
// roundings repeat, so the output is off by, in rms, for scores of a standard
// deviation of 0.7, 1.5, 2.5, 5 and 10 (4096 tokens; 32768 the same within a
// tenth): 0.44e-3, 0.94e-3, 1.05e-3, 1.4e-3 and 1.7e-3 of its size; FP8 keys,
// which fp16 holds exactly, 0.30e-3 to 0.75e-3.  A bf16 output's own rounding
// is 1.65e-3, an fp16 one's 0.21e-3: only bf16 outputs come here
// (prefix_attention).
//
// m is a lazy reference: it moves (and l and O are rescaled) only when a weight
// exceeds 2^15, half of what fp16 holds.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "tqb_common.cuh"
#include "tqb_internal.h"
#include "tqb_umma.cuh"

namespace tqb {

// Kernels that gave up a wait (read by tqb_wait_timeouts).
__device__ unsigned int g_prefix_timeouts = 0;

namespace {

constexpr int kTile = 128;                       // tokens of a tile, rows of a stream
constexpr int kTilePages = kTile / kBlockSize;   // 8
constexpr int kOperand = kTile * kHeadDim * 2;   // 32 KB: one fp16 operand tile
constexpr int kHalf = kOperand / 2;              // 16 KB: its 64-element half
constexpr int kQOff = 0, kKOff = 2 * kOperand, kVOff = 4 * kOperand, kLutOff = 6 * kOperand;
constexpr int kAuxOff = kLutOff + 256 * 32 * 4;  // the K table: 256 entries, a copy per lane
constexpr int kBarOff = kAuxOff + 2 * kTile * 4;
constexpr int kPrefixSmem = kBarOff + 192;
static_assert(kPrefixSmem <= 232448, "shared memory per CTA");
constexpr int kSoftmaxWarps = 8, kProducerWarps = 4;
constexpr int kPrefixThreads = (kSoftmaxWarps + kProducerWarps) * 32;  // whole warpgroups
// Registers per thread: 168 at the launch (the most that 384 threads can
// have), moved between the warpgroups by setmaxnreg (the shares add up to the
// launch's).
constexpr int kPrefixRegs = 168, kSoftmaxRegs = 200, kProducerRegs = 104;
static_assert(2 * kSoftmaxRegs + kProducerRegs <= 3 * kPrefixRegs && kPrefixRegs * kPrefixThreads <= 65536, "register split");
// A row's largest weight stands at 2^7 where its reference is set and may grow
// to 2^15 before it moves again (weighing a tile twice: 2^8 and 2^15 take 5 us
// more at 64 x 32768).  fp16 ends at 2^-25, so weights down to 2^-32 of the
// largest count, and those above 2^-21 of it have all their bits: a first
// token that takes nearly all of the weight leaves the others theirs.
constexpr float kStart = 7.0f, kMost = 32768.0f;

// Barriers (8 bytes each) at kBarOff, then words.
// Two of each: stages of K and V, S and the last products (after an error) per
// stream.
enum : uint32_t { kKFull = 0, kVFull = 16, kKEmpty = 32, kVEmpty = 48, kSFull = 64, kDone = 80, kMasks = 96, kTmem = 112,
                  kAbort = 116 };


__device__ __forceinline__ uint32_t dup16(uint32_t h) { return __byte_perm(h, 0u, 0x1010); }
__device__ __forceinline__ uint32_t hmul2u(uint32_t a, uint32_t b) { return h2_as_u32(__hmul2(u32_as_h2(a), u32_as_h2(b))); }
__device__ __forceinline__ uint32_t g16(const uint8_t* p) { return __ldg(reinterpret_cast<const unsigned short*>(p)); }
__device__ __forceinline__ uint32_t g32(const uint8_t* p) { return __ldg(reinterpret_cast<const unsigned int*>(p)); }
__device__ __forceinline__ uint4 g128(const uint8_t* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }
__device__ __forceinline__ uint32_t g2x16(const uint8_t* p) { return g16(p) | (g16(p + 2) << 16); }
template <bool A2>  // four bytes, 2-byte aligned (A2) or 4-byte aligned
__device__ __forceinline__ uint32_t gw(const uint8_t* p) { return A2 ? g2x16(p) : g32(p); }

// Codes and metadata of one token's 32 dims [32c, 32c + 32).
template <int L>
struct RawK {
    uint32_t k[layout_fp8_keys(L) ? 8 : 4], norm;
};
struct RawV {
    uint32_t v[4], scale, zero;
};
// Addresses of a token-head's key codes, value codes and metadata.
template <int L>
struct Where {
    const uint8_t *k, *v, *norm, *scale, *zero;
    __device__ __forceinline__ Where(const PrefixParams& P, int id, uint32_t off, uint32_t h) {
        constexpr bool k8 = layout_fp8_keys(L);
        constexpr int kKey = aos_key_bytes(L), kRow = kKey + val_code_bytes(L);
        const uint8_t* base = P.cache + (size_t)(uint32_t)id * (size_t)P.block_bytes;
        if constexpr (layout_is_aos(L)) {
            k = base + (size_t)off * P.pos_stride + (size_t)h * P.head_stride;
            v = k + aos_val_off(L);
            norm = k + aos_norm_off(L);
            scale = k + aos_scale_off(L);
            zero = scale + 2;
        } else {
            constexpr uint32_t kFields = k8 ? 2 : 3;
            k = base + off * ((uint32_t)P.Hk * kRow) + h * (uint32_t)kRow;
            v = k + kKey;
            norm = base + (uint32_t)kBlockSize * P.Hk * kRow + (h * kFields * kBlockSize + off) * 2;
            scale = norm + (kFields - 2) * kBlockSize * 2;
            zero = scale + kBlockSize * 2;
        }
    }
};
// A page that does not exist (id < 0) reads as zeros; the mask hides its scores.
template <int L>
__device__ __forceinline__ void load_k(RawK<L>& r, const PrefixParams& P, int id, uint32_t off, uint32_t h, uint32_t c) {
    constexpr bool k8 = layout_fp8_keys(L), k3 = layout_3bit_keys(L), aos = layout_is_aos(L);
    constexpr int kWords = k8 ? 8 : k3 ? 3 : 4;
    if (id < 0) {
#pragma unroll
        for (int i = 0; i < kWords; i++) r.k[i] = 0u;
        r.norm = 0u;
        return;
    }
    const Where<L> w(P, id, off, h);
    const uint8_t* p = w.k + 4 * kWords * c;
    if constexpr (!aos && !k3) {
#pragma unroll
        for (int i = 0; i < kWords; i += 4) {
            const uint4 a = g128(p + 4 * i);
            r.k[i] = a.x; r.k[i + 1] = a.y; r.k[i + 2] = a.z; r.k[i + 3] = a.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kWords; i++) r.k[i] = gw<aos>(p + 4 * i);
    }
    r.norm = k8 ? 0u : g16(w.norm);
}
template <int L>
__device__ __forceinline__ void load_v(RawV& r, const PrefixParams& P, int id, uint32_t off, uint32_t h, uint32_t c) {
    constexpr bool v3 = layout_3bit_values(L), aos = layout_is_aos(L);
    if (id < 0) {
        r.v[0] = r.v[1] = r.v[2] = r.v[3] = r.scale = r.zero = 0u;
        return;
    }
    const Where<L> w(P, id, off, h);
    const uint8_t* p = w.v + (v3 ? 12 : 16) * c;
    if constexpr (!aos && !v3) {
        const uint4 a = g128(p);
        r.v[0] = a.x; r.v[1] = a.y; r.v[2] = a.z; r.v[3] = a.w;
    } else {
#pragma unroll
        for (int i = 0; i < (v3 ? 3 : 4); i++) r.v[i] = gw<aos>(p + 4 * i);
    }
    r.scale = g16(w.scale);
    r.zero = g16(w.zero);
}
// 3-bit codes 8i .. 8i + 7 (24 bits) of a 12-byte run.
__device__ __forceinline__ uint32_t bits24(const uint32_t* w, int i) {
    return i == 0 ? w[0] & 0xFFFFFFu
         : i == 1 ? __funnelshift_r(w[0], w[1], 24) & 0xFFFFFFu
         : i == 2 ? __funnelshift_r(w[1], w[2], 16) & 0xFFFFFFu
                  : w[2] >> 8;
}

// 32 dims of a token into the K tile: 4 16-byte chunks of its row.
template <int L>
__device__ __forceinline__ void put_k(uint8_t* smem, uint32_t tile, const RawK<L>& r, uint32_t tok, uint32_t c, int lane) {
    constexpr bool k8 = layout_fp8_keys(L), k3 = layout_3bit_keys(L), aos = layout_is_aos(L);
    uint32_t f[16];
    if constexpr (k8) {
#pragma unroll
        for (int i = 0; i < 16; i++) f[i] = fp8x2_to_h2((r.k[i >> 1] >> (16 * (i & 1))) & 0xFFFFu);
    } else {
        const uint8_t* lut = smem + kLutOff + 4 * lane;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            uint32_t at;  // entry (two codes) * 128 bytes
            const int j = i & 3;
            if constexpr (k3) {
                const uint32_t x = bits24(r.k, i >> 2);
                at = (j == 0 ? x << 7 : j == 1 ? x << 1 : j == 2 ? x >> 5 : x >> 11) & 0x1F80u;
            } else {
                const uint32_t x = r.k[i >> 2];
                at = (j == 0 ? x << 7 : j == 1 ? x >> 1 : j == 2 ? x >> 9 : x >> 17) & 0x7F80u;
            }
            f[i] = *reinterpret_cast<const uint32_t*>(lut + at);
        }
        uint32_t norm = r.norm;
        if constexpr (aos) {
            // AoS stores the raw |k|: divide by the centroids' length (the
            // token's four quarters sit 8 lanes apart)
            float q = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float2 x = __half22float2(u32_as_h2(f[i]));
                q = fmaf(x.x, x.x, fmaf(x.y, x.y, q));
            }
            q += __shfl_xor_sync(0xffffffffu, q, 8);
            q += __shfl_xor_sync(0xffffffffu, q, 16);
            norm = __half_as_ushort(__float2half_rn(half_bits_to_float(norm) * rsqrtf(q + 1e-16f)));
        }
        const uint32_t n2 = dup16(norm);
#pragma unroll
        for (int i = 0; i < 16; i++) f[i] = hmul2u(f[i], n2);
    }
    uint8_t* row = smem + tile + (c >> 1) * kHalf + tok * 128;
#pragma unroll
    for (int i = 0; i < 4; i++)
        *reinterpret_cast<uint4*>(row + ((((c & 1) * 4 + i) ^ (tok & 7)) << 4)) =
            make_uint4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
}

// 32 dims of a token into the V tile, each group of 8 in the order 0 4 1 5 2
// 6 3 7 (the nibble pairs that one mask of a word yields): the columns of O
// come out in that order and are put right when they are written.
template <int L>
__device__ __forceinline__ void put_v(uint8_t* smem, uint32_t tile, const RawV& r, uint32_t tok, uint32_t c) {
    constexpr bool v3 = layout_3bit_values(L);
    // a nibble in the mantissa of 1024 (bits 0-3) or of 64 (bits 4-7) adds its
    // own value to it, exactly
    const __half2 k1024 = u32_as_h2(0x64006400u), k64 = u32_as_h2(0x54005400u);
    const __half2 s2 = u32_as_h2(dup16(r.scale)), z2 = u32_as_h2(dup16(r.zero));
    uint8_t* row = smem + tile + (c >> 1) * kHalf + tok * 128;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t w = v3 ? spread3to4(bits24(r.v, i)) : r.v[i];
        const uint32_t w8 = w >> 8;
        uint4 o;
        o.x = h2_as_u32(__hfma2(__hsub2(u32_as_h2(and_or(w, 0x000F000Fu, 0x64006400u)), k1024), s2, z2));
        o.y = h2_as_u32(__hfma2(__hsub2(u32_as_h2(and_or(w, 0x00F000F0u, 0x54005400u)), k64), s2, z2));
        o.z = h2_as_u32(__hfma2(__hsub2(u32_as_h2(and_or(w8, 0x000F000Fu, 0x64006400u)), k1024), s2, z2));
        o.w = h2_as_u32(__hfma2(__hsub2(u32_as_h2(and_or(w8, 0x00F000F0u, 0x54005400u)), k64), s2, z2));
        *reinterpret_cast<uint4*>(row + ((((c & 1) * 4 + i) ^ (tok & 7)) << 4)) = o;
    }
}

// Where a CTA works: its n tiles from t0 on and rows [row0, row0 + rows), and
// the tiles of a stream (every tile, or with `split` every other one).
struct Place {
    int h, t0, n, row0, rows;
    bool split;
    __device__ __forceinline__ int steps(int m) const { return split ? (n + 1 - m) / 2 : (m == 0 || rows > kTile ? n : 0); }
    __device__ __forceinline__ int tile(int m, int u) const { return split ? 2 * u + m : u; }  // from t0 on
};

template <int L>
__device__ __forceinline__ void dequantise(const PrefixParams& P, const Place& W, uint8_t* smem, uint32_t bars, volatile uint32_t* abort,
                           int pw, int lane) {
    const uint32_t t8 = lane & 7, c = lane >> 3;
    const uint32_t off = (pw & 1) * 8 + t8;  // token in its page
    const int nblocks = P.num_blocks > 0 && P.num_blocks < 0x7fffffff ? (int)P.num_blocks : 0x7fffffff;
    // Task i of a tile: token 32i + 8 pw + t8, in page 2i + pw / 2.
    auto page_id = [&](int tile, int i) {
        const int pg = (W.t0 + tile) * kTilePages + 2 * i + (pw >> 1);
        if (tile >= W.n || pg >= P.n_pages) return -1;
        const int id = __ldg(P.pages + pg);
        return id >= 0 && id < nblocks ? id : -1;
    };
    // The codes of the next tile are in flight while this one is unpacked.
    RawK<L> rk[4];
    RawV rv[4];
    int ids[4], next[4];
#pragma unroll
    for (int i = 0; i < 4; i++) ids[i] = page_id(0, i);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        load_k<L>(rk[i], P, ids[i], off, W.h, c);
        next[i] = page_id(1, i);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) load_v<L>(rv[i], P, ids[i], off, W.h, c);
    for (int j = 0; j < W.n; j++) {
        const int s = j & 1;
        const uint32_t phase = ((j >> 1) & 1) ^ 1;
        if (!bar_wait_warp(bars + kKEmpty + 8 * s, phase, abort)) return;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            put_k<L>(smem, kKOff + s * kOperand, rk[i], 32 * i + 8 * pw + t8, c, lane);
            load_k<L>(rk[i], P, next[i], off, W.h, c);
        }
        // pages of this tile that exist, a bit each (warps 0 and 2 own four)
        if ((pw & 1) == 0 && lane == 0) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) m |= ids[i] >= 0 ? 1u << (2 * i + (pw >> 1)) : 0u;
            smem[kBarOff + kMasks + 4 * (j & 3) + (pw >> 1)] = (uint8_t)m;
        }
        fence_async_smem();
        bar_arrive(bars + kKFull + 8 * s);
        if (!bar_wait_warp(bars + kVEmpty + 8 * s, phase, abort)) return;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            put_v<L>(smem, kVOff + s * kOperand, rv[i], 32 * i + 8 * pw + t8, c);
            ids[i] = next[i];
            load_v<L>(rv[i], P, ids[i], off, W.h, c);
            next[i] = page_id(j + 2, i);
        }
        fence_async_smem();
        bar_arrive(bars + kVFull + 8 * s);
    }
}

// The products of a stream, issued by its first warp (converged).  They execute
// in the order of issue, so the scores of step u + 1 may follow P V of step u on
// the same columns, and the one commit behind both (event u + 1 of the stream,
// on s_full) also says that the products up to step u are in O; event n says
// only that.
struct Products {
    uint32_t smem, bars, tmem, m;
    volatile uint32_t* abort;
    const Place& W;

    // The operands of step u's products: its values, the next step's keys.
    // Waited for ahead of the scores, off the way from weights to scores.
    __device__ __forceinline__ bool operands(int u, int n) const {
        const int t = W.tile(m, u), t1 = W.tile(m, u + 1);
        return bar_wait_warp(bars + kVFull + 8 * (t & 1), (t >> 1) & 1, abort) &&
               (u + 1 == n || bar_wait_warp(bars + kKFull + 8 * (t1 & 1), (t1 >> 1) & 1, abort));
    }
    __device__ __forceinline__ void scores(int u) const {  // S = Q K^T of step u
        constexpr uint32_t kQK = umma_idesc(kTile, kTile, false);
        const uint64_t q = umma_desc(smem + kQOff + (W.split ? 0 : m * kOperand), 16, 1024);
        const uint64_t k = umma_desc(smem + kKOff + (W.tile(m, u) & 1) * kOperand, 16, 1024);
#pragma unroll
        for (int e = 0; e < 8; e++) {  // 16 dims: 32 bytes of a swizzled row, the upper 64 dims a half further
            const uint64_t at = ((e >> 2) * kHalf + (e & 3) * 32) >> 4;
            umma_ss(tmem + m * kTile, q + at, k + at, kQK, e != 0);
        }
    }
    __device__ __forceinline__ bool begin() const {
        const int s = W.tile(m, 0) & 1;
        if (!bar_wait_warp(bars + kKFull + 8 * s, 0, abort)) return false;
        tc_fence_after();
        scores(0);
        umma_commit(bars + kSFull + 8 * m);
        umma_commit(bars + kKEmpty + 8 * s);
        return true;
    }
    __device__ __forceinline__ void step(int u, int n) const {  // O += P V of step u, S of step u + 1
        constexpr uint32_t kPV = umma_idesc(kTile, kHeadDim, true);
        const int s = W.tile(m, u) & 1;
        tc_fence_after();
        const uint64_t v = umma_desc(smem + kVOff + s * kOperand, kHalf, 1024);
#pragma unroll
        for (int e = 0; e < 8; e++)  // 16 tokens: two 8-row groups
            umma_ts(tmem + 2 * kTile + m * kHeadDim, tmem + m * kTile + 8 * e, v + e * (2048 >> 4), kPV, u != 0 || e != 0);
        if (u + 1 < n) scores(u + 1);
        umma_commit(bars + kSFull + 8 * m);
        umma_commit(bars + kVEmpty + 8 * s);
        if (u + 1 < n) umma_commit(bars + kKEmpty + 8 * (W.tile(m, u + 1) & 1));
    }
};

// Running reference and sum of a row.
struct RowState {
    float ref, l;
};

// Moves the reference of the rows whose exponents exceed it by too much, and
// scales what they have summed so far: l and O (whose earlier products are in
// it since these scores were announced).  Rare.
__device__ __noinline__ RowState raise(RowState st, float top, bool over, uint32_t to, bool has_o) {
    const float f = over ? ex2_approx(-top) : 1.0f;
    if (over) st.ref += top;
    st.l *= f;
    if (has_o) {
        for (int i = 0; i < kHeadDim; i += 16) {
            uint32_t o[16];
            tmem_ld16(o, to + i);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 16; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
            tmem_st16(to + i, o);
        }
        tmem_wait_st();
    }
    return st;
}

// The largest score of this thread's row (rare: from TMEM again).
template <bool MASK>
__device__ __noinline__ float largest(uint32_t ts, int lim, uint32_t pages) {
    float top = -INFINITY;
    for (int q = 0; q < kTile; q += 16) {
        uint32_t s[16];
        tmem_ld16(s, ts + q);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 16; j++)
            if (!MASK || (q + j < lim && (pages >> (q >> 4)) & 1u)) top = fmaxf(top, __uint_as_float(s[j]));
    }
    return top;
}

// A tile's scores of this thread's row turned into weights p = exp2(s kfac -
// ref) in their place (columns 0 .. 63, two fp16 each).  The whole row is in
// registers, and nothing stands before the exponentials: whether the reference
// still holds is read off the weights (their largest, infinite where fp16 ends),
// and the scores are weighed again where it does not.
template <bool MASK>
__device__ __forceinline__ void weigh(RowState& st, uint32_t ts, uint32_t to, bool has_o, float kfac, int lim,
                                      uint32_t pages) {
    const uint64_t k2 = pack2(kfac, kfac);
    if (__any_sync(0xffffffffu, st.ref == -INFINITY)) {  // rows that see their first tokens
        const float top = largest<MASK>(ts, lim, pages);
        if (st.ref == -INFINITY && top < INFINITY) st.ref = top * kfac - kStart;
    }
    for (;;) {
        uint32_t s[4][32], p[64];
#pragma unroll
        for (int q = 0; q < 4; q++) tmem_ld32(s[q], ts + 32 * q);
        tmem_wait_ld();
        const float r = st.ref == -INFINITY ? 0.0f : st.ref;
        const uint64_t r2 = pack2(-r, -r);
        uint64_t acc = pack2(0.0f, 0.0f);
        __half2 most = u32_as_h2(0u);
#pragma unroll
        for (int q = 0; q < 4; q++)
#pragma unroll
            for (int j = 0; j < 16; j++) {
                uint64_t x = fma2((uint64_t)s[q][2 * j] | ((uint64_t)s[q][2 * j + 1] << 32), k2, r2);
                if constexpr (MASK) {
                    const int t = 32 * q + 2 * j;
                    const bool page = (pages >> (t >> 4)) & 1u;
                    x = pack2(page && t < lim ? lo2(x) : -INFINITY, page && t + 1 < lim ? hi2(x) : -INFINITY);
                }
                const float a = ex2_approx(lo2(x)), b = ex2_approx(hi2(x));
                acc = add2(acc, pack2(a, b));
                const __half2 h = __floats2half2_rn(a, b);
                most = __hmax2(most, h);
                p[16 * q + j] = h2_as_u32(h);
            }
        const bool over = fmaxf(__low2float(most), __high2float(most)) > kMost;
        if (__any_sync(0xffffffffu, over)) {
            const float x = largest<MASK>(ts, lim, pages) * kfac - r - kStart;
            const bool move = over && x > 0.0f && x < INFINITY;  // infinite scores stay as they are
            if (__any_sync(0xffffffffu, move)) {
                st = raise(st, x, move, to, has_o);
                continue;
            }
        }
        st.l += lo2(acc) + hi2(acc);
        tmem_st32(ts, p);
        tmem_st32(ts + 32, p + 32);
        tmem_wait_st();
        return;
    }
}

__device__ __forceinline__ void softmax(const PrefixParams& P, const Place& W, uint8_t* smem, uint32_t smem_base, uint32_t bars, uint32_t tmem,
                        volatile uint32_t* abort, int m, int warp, int lane) {
    const int wq = warp & 3;
    const uint32_t lanes = (uint32_t)(32 * wq) << 16;
    const uint32_t ts = tmem + lanes + m * kTile, to = tmem + lanes + 2 * kTile + m * kHeadDim;
    const int local = (W.split ? 0 : m * kTile) + 32 * wq + lane;  // row of the CTA
    const bool live = local < W.rows;
    const int row = W.row0 + min(local, W.rows - 1);
    const int b = (int)P.div_g.div((uint32_t)row), g = row - b * P.G;
    const float kfac = *reinterpret_cast<const float*>(smem + kAuxOff + 4 * ((W.split ? 0 : m * kTile) + 32 * wq + lane));
    // tokens of the chunk this row sees, from the chunk's start
    const int lim = max(min(__ldg(P.seq_lens + b), P.n_pages * kBlockSize), 0) - W.t0 * kTile;
    const bool any_row = __any_sync(0xffffffffu, live);
    // (a row that sees nothing of the chunk has weights of zero at any reference)
    RowState st{lim > 0 ? -INFINITY : 0.0f, 0.0f};
    const int n = W.steps(m);
    const Products mma{smem_base, bars, tmem, (uint32_t)m, abort, W};
    bool ok = true;
    if (n > 0 && wq == 0) ok = mma.begin();
    // The streams take turns at weighing: on their own they fall into step,
    // both weighing (sharing the exponential units) and then both waiting for
    // their products; in turns one's products run under the other's weighing.
    // Stream m's steps are its turns on barrier 5 + m, stream 0 first (its
    // count of steps is stream 1's or one more).
    const int other = W.steps(1 - m);
    const bool turns = n > 0 && other > 0;
    if (turns && m == 1) asm volatile("bar.arrive 5, 256;\n" ::: "memory");
    for (int u = 0; u < n; u++) {  // every warp takes every turn at the barrier, also when a wait has given up
        const int tile = W.tile(m, u);
        if (wq == 0) ok = ok && mma.operands(u, n);
        ok = ok && bar_wait_warp(bars + kSFull + 8 * m, u & 1, abort);
        tc_fence_after();
        if (turns) asm volatile("bar.sync %0, 256;\n" ::"r"(5 + m) : "memory");
        if (ok && any_row) {
            const uint32_t pages = smem[kBarOff + kMasks + 4 * (tile & 3)] | smem[kBarOff + kMasks + 4 * (tile & 3) + 1];
            const int left = lim - tile * kTile;
            if (__any_sync(0xffffffffu, left < kTile || pages != 0xFFu))
                weigh<true>(st, ts, to, u > 0, kfac, left, pages);
            else
                weigh<false>(st, ts, to, u > 0, kfac, left, pages);
        }
        if (u + m < other) asm volatile("bar.arrive %0, 256;\n" ::"r"(6 - m) : "memory");
        tc_fence_before();
        asm volatile("bar.sync %0, 128;\n" ::"r"(3 + m) : "memory");  // the stream's weights are complete
        if (wq == 0 && ok) mma.step(u, n);
    }
    // ---- the partial rows ----
    // (also: every product has ended before the CTA frees its TMEM)
    if (n > 0 && !(ok && bar_wait_warp(bars + kSFull + 8 * m, n & 1, abort))) {
        if (wq == 0) {  // what has been issued ends first, if it ends
            umma_commit(bars + kDone + 8 * m);
            bar_wait_warp(bars + kDone + 8 * m, 0, nullptr);
        }
        return;
    }
    tc_fence_after();
    if (!any_row) return;
    const int sp = W.split ? 2 * (int)blockIdx.x + m : (int)blockIdx.x;
    const bool seen = st.l > 0.0f || st.l != st.l;
    const float inv = seen ? rcp_approx(st.l) : 0.0f;
    float* dst = P.mid + (int64_t)b * P.msb + (int64_t)(W.h * P.G + g) * P.msh + (int64_t)sp * P.mss;
    const uint32_t live_rows = __ballot_sync(0xffffffffu, live);
    if (live) dst[kHeadDim] = seen ? (st.ref + lg2_approx(st.l)) * kLn2 : -INFINITY;
    // 32 x 32 blocks turn through shared memory (this stream's query tile, or
    // the unused second one; 16-byte chunk c of row r at chunk c ^ (r & 7)), so
    // that rows are written in runs of 128 bytes: four rows per 16-byte store
    // where the rows are aligned (the partials' pitch is the caller's), one per
    // 4-byte store otherwise.
    uint8_t* turn = smem + kQOff + (W.split ? kOperand + m * kHalf : m * kOperand) + wq * 4096;
    const bool vec = ((reinterpret_cast<uintptr_t>(P.mid) & 15) | ((P.msb | P.msh | P.mss) & 3)) == 0;
    const unsigned long long mine = reinterpret_cast<unsigned long long>(dst);
    float* rows[8];
    if (vec) {
#pragma unroll
        for (int i = 0; i < 8; i++)
            rows[i] = reinterpret_cast<float*>(__shfl_sync(0xffffffffu, mine, 4 * i + (lane >> 3))) + 4 * (lane & 7);
    }
#pragma unroll 1
    for (int q = 0; q < 4; q++) {
        uint32_t o[32];
        if (n > 0) {
            tmem_ld32(o, to + 32 * q);
            tmem_wait_ld();
        }
#pragma unroll
        for (int c = 0; c < 8; c++) {  // dims 4c .. 4c + 3: every other column of the group of 8, from c & 1 on
            float v[4];
#pragma unroll
            for (int j = 0; j < 4; j++)
                v[j] = seen ? __uint_as_float(o[(c >> 1) * 8 + 2 * j + (c & 1)]) * inv : 0.0f;
            *reinterpret_cast<float4*>(turn + 128 * lane + ((c ^ (lane & 7)) << 4)) = make_float4(v[0], v[1], v[2], v[3]);
        }
        __syncwarp();
        if (vec) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int r = 4 * i + (lane >> 3);
                const float4 v = *reinterpret_cast<const float4*>(turn + 128 * r + (((lane & 7) ^ (r & 7)) << 4));
                if ((live_rows >> r) & 1u) *reinterpret_cast<float4*>(rows[i] + 32 * q) = v;
            }
        } else {
            for (int r = 0; r < 32; r++) {
                float* to_row = reinterpret_cast<float*>(__shfl_sync(0xffffffffu, mine, r));
                const float v = *reinterpret_cast<const float*>(turn + 128 * r + ((((lane >> 2) ^ (r & 7)) << 4) | ((lane & 3) << 2)));
                if ((live_rows >> r) & 1u) to_row[32 * q + lane] = v;
            }
        }
        __syncwarp();
    }
}

// K table: entry = two codes, {c[low], c[high]} in fp16, a copy per lane.  A
// producer warp makes 64 entries (16 for 3-bit codes), a lane each or two, and
// spreads them over the copies.
template <int L>
__device__ __forceinline__ void build_table(const PrefixParams& P, uint8_t* smem, int pw, int lane) {
    constexpr bool k3 = layout_3bit_keys(L);
    constexpr int kPairs = k3 ? 64 : 256, kBits = k3 ? 3 : 4, kMask = k3 ? 7 : 15, kMine = kPairs / kProducerWarps;
#pragma unroll
    for (int e0 = 0; e0 < kMine; e0 += 16) {
        const int pair = kMine * pw + e0 + (lane & 15);
        const uint32_t v = h2_as_u32(__floats2half2_rn(__ldg(P.cents + (pair & kMask)), __ldg(P.cents + (pair >> kBits))));
        uint32_t* lut = reinterpret_cast<uint32_t*>(smem + kLutOff) + (kMine * pw + e0) * 32 + lane;
#pragma unroll
        for (int i = 0; i < 16; i++) lut[32 * i] = __shfl_sync(0xffffffffu, v, i);
    }
}

// Queries: fp16, scaled per row into [2^14, 2^15), 128-byte swizzle, and the
// rows' score factors.  A softmax warp takes rows warp, warp + 8, ..., 16 of
// them in flight.
__device__ __forceinline__ void load_queries(const PrefixParams& P, const Place& W, uint8_t* smem, int warp, int lane) {
    const int slots = W.split || W.rows <= kTile ? kTile : 2 * kTile;
    for (int r0 = warp; r0 < slots; r0 += 16 * kSoftmaxWarps) {
        float4 x[16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int r = r0 + i * kSoftmaxWarps;
            x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (r < W.rows) {
                const int row = W.row0 + r, b = (int)P.div_g.div((uint32_t)row), g = row - b * P.G;
                x[i] = __ldg(reinterpret_cast<const float4*>(P.q + (int64_t)b * P.qsb + (int64_t)(W.h * P.G + g) * P.qsh) + lane);
            }
        }
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int r = r0 + i * kSoftmaxWarps;
            // (bits of non-negative floats order as the floats do)
            const float amax = __uint_as_float(__reduce_max_sync(
                0xffffffffu,
                __float_as_uint(fmaxf(fmaxf(fabsf(x[i].x), fabsf(x[i].y)), fmaxf(fabsf(x[i].z), fabsf(x[i].w))))));
            const int e = fp16_scale_exp(amax);
            const float f = exp2i(e);
            if (lane == 0) reinterpret_cast<float*>(smem + kAuxOff)[r] = P.scale * kLog2e * exp2i(-e);
            // dims 4 lane .. 4 lane + 3: half lane / 16, chunk (lane % 16) / 2
            uint8_t* at = smem + kQOff + (r >> 7) * kOperand + (lane >> 4) * kHalf + (r & 127) * 128 +
                          ((((lane & 15) >> 1) ^ (r & 7)) << 4) + (lane & 1) * 8;
            *reinterpret_cast<uint2*>(at) = make_uint2(h2_as_u32(__floats2half2_rn(x[i].x * f, x[i].y * f)),
                                                       h2_as_u32(__floats2half2_rn(x[i].z * f, x[i].w * f)));
        }
    }
}

template <int L>
__global__ void __launch_bounds__(kPrefixThreads, 1) prefix_kernel(const PrefixParams P) {
    extern __shared__ __align__(1024) uint8_t smem[];
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const uint32_t base = smem_addr(smem), bars = base + kBarOff;
    volatile uint32_t* abort = reinterpret_cast<volatile uint32_t*>(smem + kBarOff + kAbort);
    pdl_trigger();

    Place W;
    const int R = P.B * P.G, n_tiles = (P.n_pages + kTilePages - 1) / kTilePages;
    W.h = blockIdx.y;
    W.t0 = (int)((int64_t)n_tiles * blockIdx.x / gridDim.x);
    W.n = (int)((int64_t)n_tiles * (blockIdx.x + 1) / gridDim.x) - W.t0;
    W.row0 = blockIdx.z * 2 * kTile;
    W.rows = min(R - W.row0, 2 * kTile);
    W.split = P.split != 0;

    if (tid == 0) {
        const int readers = !W.split && W.rows > kTile ? 2 : 1;  // streams that read each stage
        for (int s = 0; s < 2; s++) {
            bar_init(bars + kKFull + 8 * s, kProducerWarps * 32);
            bar_init(bars + kVFull + 8 * s, kProducerWarps * 32);
            bar_init(bars + kKEmpty + 8 * s, readers);
            bar_init(bars + kVEmpty + 8 * s, readers);
            bar_init(bars + kSFull + 8 * s, 1);
            bar_init(bars + kDone + 8 * s, 1);
        }
        *abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == kSoftmaxWarps) tmem_alloc<512>(bars + kTmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_wait();  // the rotated queries, and the kernel before that reads mid_o

    // All 512 columns start at column 0: a constant, so that the MMAs' TMEM
    // operands need no register (checked, as an error that ends the waits).
    constexpr uint32_t tmem = 0;
    if (tid == 0 && *reinterpret_cast<volatile uint32_t*>(smem + kBarOff + kTmem) != tmem) *abort = 1;

    if (warp < kSoftmaxWarps) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kSoftmaxRegs));
        load_queries(P, W, smem, warp, lane);
        fence_async_smem();
        asm volatile("bar.sync 1, %0;\n" ::"n"(kSoftmaxWarps * 32) : "memory");  // queries and score factors
        softmax(P, W, smem, base, bars, tmem, abort, warp >> 2, warp, lane);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kProducerRegs));
        if constexpr (!layout_fp8_keys(L)) {
            build_table<L>(P, smem, warp - kSoftmaxWarps, lane);
            asm volatile("bar.sync 2, %0;\n" ::"n"(kProducerWarps * 32) : "memory");
        }
        dequantise<L>(P, W, smem, bars, abort, warp - kSoftmaxWarps, lane);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kSoftmaxWarps) tmem_free<512>(*reinterpret_cast<volatile uint32_t*>(smem + kBarOff + kTmem));
    if (tid == 0 && *abort != 0) atomicAdd(&g_prefix_timeouts, 1u);
}

template <int L>
int launch_prefix_t(const PrefixParams& P, cudaStream_t stream) {
    auto kern = prefix_kernel<L>;
    static thread_local int configured_dev = -1;
    int dev = 0;
    cudaGetDevice(&dev);
    if (configured_dev != dev) {
        // the register split draws on what the kernel was launched with
        cudaFuncAttributes a{};
        if (cudaFuncGetAttributes(&a, kern) != cudaSuccess) return report_launch(cudaGetLastError());
        if (a.numRegs < kPrefixRegs) {
            set_error_detail("the shared-prefix kernel was built with fewer registers than its split needs");
            return TQB_ERR_UNSUPPORTED;
        }
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kPrefixSmem) != cudaSuccess)
            return report_launch(cudaGetLastError());
        configured_dev = dev;
    }
    const unsigned blocks = (unsigned)(((int64_t)P.B * P.G + 2 * kTile - 1) / (2 * kTile));
    return report_launch(launch_pdl(kern, dim3((unsigned)P.chunks, (unsigned)P.Hk, blocks), dim3(kPrefixThreads), kPrefixSmem,
                                    stream, P));
}

}  // namespace

int launch_prefix(const PrefixParams& P, cudaStream_t stream) {
    switch (P.layout) {
        case TQB_LAYOUT_SOA: return launch_prefix_t<TQB_LAYOUT_SOA>(P, stream);
        case TQB_LAYOUT_SOA_K8: return launch_prefix_t<TQB_LAYOUT_SOA_K8>(P, stream);
        case TQB_LAYOUT_SOA_K3: return launch_prefix_t<TQB_LAYOUT_SOA_K3>(P, stream);
        case TQB_LAYOUT_SOA_K3V3: return launch_prefix_t<TQB_LAYOUT_SOA_K3V3>(P, stream);
        case TQB_LAYOUT_AOS: return launch_prefix_t<TQB_LAYOUT_AOS>(P, stream);
        case TQB_LAYOUT_AOS_K8: return launch_prefix_t<TQB_LAYOUT_AOS_K8>(P, stream);
        case TQB_LAYOUT_AOS_K3: return launch_prefix_t<TQB_LAYOUT_AOS_K3>(P, stream);
        case TQB_LAYOUT_AOS_K3V3: return launch_prefix_t<TQB_LAYOUT_AOS_K3V3>(P, stream);
        default: return TQB_ERR_INVALID_ARG;
    }
}

int read_prefix_timeouts(unsigned int* count, bool reset) {
    cudaError_t e = cudaMemcpyFromSymbol(count, g_prefix_timeouts, sizeof(unsigned int));
    if (e == cudaSuccess && reset) {
        const unsigned int zero = 0;
        e = cudaMemcpyToSymbol(g_prefix_timeouts, &zero, sizeof(unsigned int));
    }
    return e == cudaSuccess ? TQB_OK : report_launch(e);
}

}  // namespace tqb
