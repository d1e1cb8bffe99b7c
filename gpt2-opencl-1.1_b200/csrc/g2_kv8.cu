// g2_kv8.cu -- a paged KV cache of 8-bit codes with one scale for each page
// (block of tokens) and head: writing rows (g2k_kv8_append), reading them back
// (g2k_kv8_gather) and attention over it (g2k_kv8_attention).
//
// The value of a code c on a page with scale s is c s.  Codes are int8
// (-127..127) or e4m3 (up to 448).
#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>

#include "g2_args.h"
#include "g2_device.cuh"
#include "g2_mma.cuh"

namespace g2 {

namespace {

struct Rows8 {   // which rows a call is about (see gpt2b200.h)
    int n_rows, n_seq, max_q;
    const int *q_start;
    const int *table;
    int table_stride;
    int *status;
};

struct Span {
    int first, n;   // rows of the sequence; n = -1: out of range
};

__device__ __forceinline__ void bad(const Rows8 &r) {
    if (r.status) atomicExch(r.status, G2_ERR_RANGE);
}

__device__ __forceinline__ Span seq_rows(const Rows8 &r, int s) {
    Span p{s, 1};
    if (r.q_start) {
        const int next = r.q_start[s + 1];
        p.first = r.q_start[s];
        const long long n = (long long)next - p.first;
        if (n < 0 || n > r.max_q || p.first < 0 || p.first + n > r.n_rows) {
            bad(r);
            return Span{0, -1};
        }
        p.n = (int)n;
    }
    return p;
}

__device__ __forceinline__ int page_of(const Rows8 &r, const g2_kv8 &c, int s, int block) {
    const int page = r.table[(long long)s * r.table_stride + block];
    if (page >= 0 && page < c.n_pages) return page;
    bad(r);
    return -1;
}

// ---- codes ------------------------------------------------------------------------
constexpr float kScaleFloor = 5.421010862427522e-20f;   // 2^-64

// x / s with the last bit set when the quotient is inexact (rounding to odd), so that rounding it once
// more to 8 bits gives the nearest code of the exact quotient.  s >= 2^-64.
__device__ __forceinline__ float div_odd(float x, float s) {
    const float q = __fdiv_rn(x, s);
    const float r = __fmaf_rn(-q, s, x);
    if (r == 0.0f || q == 0.0f) return q;
    unsigned b = __float_as_uint(q);
    if ((r < 0.0f) != (q < 0.0f)) --b;   // |q| was rounded up
    return __uint_as_float(b | 1u);
}

template <int FMT>
__device__ __forceinline__ unsigned encode(float q) {
    if (FMT == G2_KV_I8) return (unsigned)max(-127, min(127, __float2int_rn(q))) & 0xffu;
    return __nv_cvt_float_to_fp8(q, __NV_SATFINITE, __NV_E4M3);
}

template <int FMT>
__device__ __forceinline__ float decode(unsigned c) {
    if (FMT == G2_KV_I8) return (float)(signed char)c;
    return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3)));
}

// The code of (code c at scale from) at scale to: the product and its quotient differ from every
// rounding border by more than a double's error unless they are on it.
template <int FMT>
__device__ __forceinline__ unsigned recode(unsigned c, float from, float to) {
    const double q = (double)decode<FMT>(c) * from / to;
    float f = __double2float_rz(q);
    if ((double)f != q) f = __uint_as_float(__float_as_uint(f) | 1u);
    return encode<FMT>(f);
}

template <typename T>
__device__ __forceinline__ float4 load4(const T *p);
template <>
__device__ __forceinline__ float4 load4<float>(const float *p) {
    return *reinterpret_cast<const float4 *>(p);
}
template <>
__device__ __forceinline__ float4 load4<__half>(const __half *p) {
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&u.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&u.y));
    return make_float4(a.x, a.y, b.x, b.y);
}

__device__ __forceinline__ unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// A block's scale after rows whose largest magnitude has the bits `peak` (integers: NaN above infinity
// above finite) join rows at scale `was` (0 where none stay).
template <int FMT>
__device__ __forceinline__ float joined_scale(unsigned peak, float was) {
    if (peak >= 0x7f800000u || was != was) return __uint_as_float(0x7fc00000u);
    return fmaxf(fmaxf(__fdiv_rn(__uint_as_float(peak), FMT == G2_KV_I8 ? 127.0f : 448.0f), kScaleFloor), was);
}

// A word of codes through the table of a magnitude's new code (rows that stay when the scale grows).
template <int FMT>
__device__ __forceinline__ unsigned recode_word(unsigned w, const unsigned char *table) {
    unsigned r = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned c = (w >> (8 * i)) & 0xffu;
        if (FMT == G2_KV_I8) {
            const int s = (int)(signed char)c, m = table[min(abs(s), 127)];
            r |= ((unsigned)(s < 0 ? -m : m) & 0xffu) << (8 * i);
        } else {
            r |= (table[c & 0x7fu] | (c & 0x80u)) << (8 * i);
        }
    }
    return r;
}

// Codes of four values at a scale whose reciprocal is `inv`.  x * inv is within 2^-22 of the quotient,
// which decides its code unless it lies that near a border; then (and for e4m3 quotients below the
// normal range) the exact quotient does: a division takes several times the product's instructions.
template <int FMT>
__device__ __forceinline__ unsigned encode4(const float4 &x, float scale, float inv) {
    const float v[4] = {x.x, x.y, x.z, x.w};
    unsigned w;
    bool near = false;
    if (FMT == G2_KV_I8) {
        constexpr float kRound = 12582912.0f;   // 1.5 * 2^23: adding it rounds to an integer in the low bits
        unsigned u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float q = fmaf(v[i], inv, kRound);
            u[i] = __float_as_uint(q);
            near |= !(fabsf(fmaf(v[i], inv, kRound - q)) < 0.4999f);   // distance from the integer; |quotient| <= 127
        }
        w = __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410);
    } else {
        float q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            q[i] = v[i] * inv;
            const unsigned b = __float_as_uint(q[i]);
            // 20 bits of an fp32 lie below the 3 of an e4m3 value: half a step is 0x80000
            near |= ((b - 0x7fff8u) & 0xfffffu) < 16u || (fabsf(q[i]) < 0.015625f && q[i] != 0.0f);
        }
        w = __nv_cvt_float2_to_fp8x2(make_float2(q[0], q[1]), __NV_SATFINITE, __NV_E4M3) |
            (unsigned)__nv_cvt_float2_to_fp8x2(make_float2(q[2], q[3]), __NV_SATFINITE, __NV_E4M3) << 16;
    }
    if (near)
        w = encode<FMT>(div_odd(v[0], scale)) | encode<FMT>(div_odd(v[1], scale)) << 8 | encode<FMT>(div_odd(v[2], scale)) << 16 |
            encode<FMT>(div_odd(v[3], scale)) << 24;
    return scale == scale ? w : 0u;
}

// ---- append -----------------------------------------------------------------------
// A *tile* is the K or V rows of one block and head.  Its new rows' largest magnitude
// gives the scale; the rows that stay are rounded again if it grew; the new rows'
// codes follow.  Bound by the rows read (2 or 4 bytes a value) and codes written.
//
// Several rows a sequence: one CTA takes the block's next tiles, as many as give a
// thread kAppendVecs 4-element loads, all in flight together: a tile by itself
// waits for its sequence's numbers, its page and its rows in turn (8 prompts of up
// to 1000 tokens of 25 heads, appended and read back: 68 us a tile at a time, 39
// with this, the encoding by a reciprocal and the gather below).
constexpr int kAppendThreads = 256, kAppendVecs = 8;

template <typename T, int FMT, int D, int VPT>
__global__ void __launch_bounds__(kAppendThreads)
    kv8_append_kernel(g2_kv8 c, const T *k, const T *v, long long stride, const int *pos, Rows8 r, int blocks_per_seq) {
    constexpr int TILES = kAppendVecs / VPT > 0 ? kAppendVecs / VPT : 1, P = VPT * 4 * kAppendThreads / D, per_row = D / 4;
    __shared__ unsigned peaks[TILES][kAppendThreads / 32];
    __shared__ float scale_s[TILES][2];                 // before, after
    __shared__ unsigned char table[TILES][128];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    pdl_wait();
    pdl_launch();
    const int s = blockIdx.x / blocks_per_seq, tile0 = blockIdx.y * TILES, n_tiles = min(TILES, 2 * c.n_kv_head - tile0);
    const int p0 = pos[s];
    const Span sp = seq_rows(r, s);
    if (sp.n <= 0) return;
    if (p0 < 0 || (long long)p0 + sp.n > (long long)r.table_stride * P) {
        bad(r);
        return;
    }
    const int block = p0 / P + blockIdx.x % blocks_per_seq;
    const long long start = (long long)block * P;
    if (start >= (long long)p0 + sp.n) return;
    const int kept = max(0, (int)(p0 - start));                        // rows 0..kept-1 stay
    const int end = (int)min((long long)P, (long long)p0 + sp.n - start);   // rows kept..end-1 are new
    const int page = page_of(r, c, s, block);                          // on its way with the rows
    const long long first = sp.first + start - p0;                     // row 0 of the block, in k and v

    float4 x[TILES][VPT];
#pragma unroll
    for (int j = 0; j < TILES; ++j) {
        const int tile = tile0 + j, h = tile >> 1;
        const T *src = (tile & 1 ? v : k) + first * stride + (long long)h * D;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int vec = t + i * kAppendThreads, row = vec / per_row;
            x[j][i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (j < n_tiles && row >= kept && row < end) x[j][i] = load4<T>(src + (long long)row * stride + (vec % per_row) * 4);
        }
    }
    if (page < 0) return;
    if (t < n_tiles) {
        const int tile = tile0 + t;
        const long long at = (long long)page * c.n_kv_head + (tile >> 1);
        scale_s[t][0] = kept > 0 ? (tile & 1 ? c.v_scale : c.k_scale)[at] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < TILES; ++j) {
        unsigned peak = 0;
#pragma unroll
        for (int i = 0; i < VPT; ++i)
            peak = max(max(peak, max(abs_bits(x[j][i].x), abs_bits(x[j][i].y))), max(abs_bits(x[j][i].z), abs_bits(x[j][i].w)));
        peak = __reduce_max_sync(0xffffffffu, peak);
        if (lane == 0) peaks[j][warp] = peak;
    }
    __syncthreads();
    bool grown = false;
    if (t < n_tiles) {
        const int tile = tile0 + t;
        const long long at = (long long)page * c.n_kv_head + (tile >> 1);
        unsigned peak = 0;
#pragma unroll
        for (int i = 0; i < kAppendThreads / 32; ++i) peak = max(peak, peaks[t][i]);
        const float to = joined_scale<FMT>(peak, scale_s[t][0]);
        scale_s[t][1] = to;
        (tile & 1 ? c.v_scale : c.k_scale)[at] = to;
        grown = kept > 0 && to > scale_s[t][0];
    }
    if (__syncthreads_or(grown)) {
        for (int i = t; i < n_tiles * 128; i += kAppendThreads) {
            const int j = i >> 7, m = i & 127;
            if (scale_s[j][1] > scale_s[j][0]) table[j][m] = (unsigned char)recode<FMT>(m, scale_s[j][0], scale_s[j][1]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < TILES; ++j) {
        if (j >= n_tiles) break;
        const int tile = tile0 + j;
        const long long at = (long long)page * c.n_kv_head + (tile >> 1);
        unsigned *dst = reinterpret_cast<unsigned *>(static_cast<unsigned char *>(tile & 1 ? c.v : c.k) + at * P * D);
        const float was = scale_s[j][0], to = scale_s[j][1], inv = __frcp_rn(to);
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int vec = t + i * kAppendThreads, row = vec / per_row;
            if (row < kept) {
                if (to > was) dst[vec] = recode_word<FMT>(dst[vec], table[j]);
            } else if (row < end) {
                dst[vec] = encode4<FMT>(x[j][i], to, inv);
            }
        }
    }
}

// One row a sequence (a decode step): one warp for each (sequence, tile).
template <typename T, int FMT, int D>
__global__ void __launch_bounds__(256) kv8_append_token_kernel(g2_kv8 c, const T *k, const T *v, long long stride, const int *pos, Rows8 r) {
    __shared__ unsigned char table[8][128];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_wait();
    pdl_launch();
    const int s = blockIdx.x, tile = blockIdx.y * 8 + warp, h = tile >> 1, P = c.page_size;
    if (tile >= 2 * c.n_kv_head) return;
    const int p = pos[s];
    const Span sp = seq_rows(r, s);
    if (sp.n <= 0) return;
    if (p < 0 || p >= (long long)r.table_stride * P) {
        bad(r);
        return;
    }
    const int page = page_of(r, c, s, p / P), kept = p & (P - 1);
    if (page < 0) return;
    const long long at = (long long)page * c.n_kv_head + h;
    unsigned *dst = reinterpret_cast<unsigned *>(static_cast<unsigned char *>(tile & 1 ? c.v : c.k) + at * P * D);
    float *scale = (tile & 1 ? c.v_scale : c.k_scale) + at;
    const float was = kept > 0 ? *scale : 0.0f;
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (lane < D / 4) x = load4<T>((tile & 1 ? v : k) + sp.first * stride + (long long)h * D + lane * 4);
    const unsigned peak = __reduce_max_sync(0xffffffffu, max(max(abs_bits(x.x), abs_bits(x.y)), max(abs_bits(x.z), abs_bits(x.w))));
    const float to = joined_scale<FMT>(peak, was);
    if (kept > 0 && to > was) {
        // the new code of each magnitude, then the rows that stay
#pragma unroll
        for (int i = 0; i < 4; ++i) table[warp][lane + 32 * i] = (unsigned char)recode<FMT>(lane + 32 * i, was, to);
        __syncwarp();
#pragma unroll 4
        for (int i = lane; i < kept * (D / 4); i += 32) dst[i] = recode_word<FMT>(dst[i], table[warp]);
    }
    if (lane < D / 4) dst[kept * (D / 4) + lane] = encode4<FMT>(x, to, __frcp_rn(to));
    if (lane == 0) *scale = to;
}

// Four codes to two fp16 pairs, exactly.  int8: code + 128 put below the exponent of 1024, minus 1152.
template <int FMT>
__device__ __forceinline__ void codes_to_half(unsigned w, unsigned &lo, unsigned &hi) {
    if (FMT == G2_KV_I8) {
        w ^= 0x80808080u;
        const __half2 off = __half2half2(__ushort_as_half((unsigned short)0x6480));   // 1152
        unsigned a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
        const __half2 x = __hsub2(*reinterpret_cast<__half2 *>(&a), off), y = __hsub2(*reinterpret_cast<__half2 *>(&b), off);
        lo = *reinterpret_cast<const unsigned *>(&x);
        hi = *reinterpret_cast<const unsigned *>(&y);
    } else {
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
            : "=r"(lo), "=r"(hi)
            : "r"(w));
    }
}

// ---- gather -----------------------------------------------------------------------
// One CTA for 16 positions of a sequence and 256 groups of four of a row's values (K
// and V), a group per thread: a thread's page and scale are the same for all its
// rows, its loads are in flight together and its stores 16 bytes (8 of fp16).
constexpr int kGatherRows = 16;

template <typename T, int FMT>
__global__ void __launch_bounds__(256)
    kv8_gather_kernel(g2_kv8 c, T *k, T *v, long long stride, const int *pos, Rows8 r, int chunks_per_seq) {
    pdl_wait();
    pdl_launch();
    const int s = blockIdx.x / chunks_per_seq;
    const int P = c.page_size, D = c.head_dim, per_row = c.n_kv_head * D / 4;
    const int p0 = pos[s];
    const Span sp = seq_rows(r, s);
    if (sp.n <= 0) return;
    if (p0 < 0 || (long long)p0 + sp.n > (long long)r.table_stride * P) {
        bad(r);
        return;
    }
    const long long base = (long long)(p0 / kGatherRows + blockIdx.x % chunks_per_seq) * kGatherRows;   // a page holds whole chunks
    const int j0 = (int)(max(base, (long long)p0) - base), j1 = (int)min((long long)kGatherRows, (long long)p0 + sp.n - base);
    if (j1 <= j0) return;
    const int page = page_of(r, c, s, (int)(base / P));
    const int q = blockIdx.y * 256 + threadIdx.x, is_v = q >= per_row, e = (is_v ? q - per_row : q) * 4;
    if (page < 0 || q >= 2 * per_row) return;
    const int h = e / D, d = e % D;
    const long long at = (long long)page * c.n_kv_head + h;
    const unsigned *src = reinterpret_cast<const unsigned *>(static_cast<const unsigned char *>(is_v ? c.v : c.k) +
                                                             (at * P + base % P) * D + d);
    const float scale = (is_v ? c.v_scale : c.k_scale)[at];
    T *dst = (is_v ? v : k) + (sp.first + base - p0) * stride + e;
    unsigned w[kGatherRows];
#pragma unroll
    for (int j = 0; j < kGatherRows; ++j)
        if (j >= j0 && j < j1) w[j] = src[j * (D / 4)];   // plain loads: the kernel before may write codes until the wait
#pragma unroll
    for (int j = 0; j < kGatherRows; ++j)
        if (j >= j0 && j < j1) {
            unsigned lo, hi;
            codes_to_half<FMT>(w[j], lo, hi);
            const float2 p = __half22float2(*reinterpret_cast<const __half2 *>(&lo)), q2 = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
            const float4 x = make_float4(p.x * scale, p.y * scale, q2.x * scale, q2.y * scale);
            if (sizeof(T) == 4) {
                *reinterpret_cast<float4 *>(dst + j * stride) = x;
            } else {
                const __half2 a = __floats2half2_rn(x.x, x.y), b = __floats2half2_rn(x.z, x.w);
                uint2 o;
                o.x = *reinterpret_cast<const unsigned *>(&a);
                o.y = *reinterpret_cast<const unsigned *>(&b);
                *reinterpret_cast<uint2 *>(dst + j * stride) = o;
            }
        }
}

// ---- attention --------------------------------------------------------------------
// out_i = sum_j w_ij c_j / sum_j w_ij / vs_j,   w_ij = 2^(t_ij - m_i),
// t_ij = (q_i . k_j) ks_j scale log2(e) + log2(vs_j),
// with k_j, c_j the integer (or e4m3) codes of a key's K and V rows and ks_j,
// vs_j the scales of its page: the V scale rides in the exponent, so a key
// costs no multiplication for either scale.
//
// A *run* is the keys of one sequence under one K/V head for a group of up to
// 4 NT query columns (column c of a sequence: row c / group, head c % group).
// Workers (WPR warps each) take whole runs where there are no more runs than workers
// and the longest is hardly longer than an equal share.  Else runs are cut into
// units of `unit` keys, and all units, in order, are shared equally, so the shares
// do not depend on how ragged the sequences are.  Beginning a run costs as much as
// several units, so each counts as `ahead` more, which hold no keys.  A run that
// crosses shares leaves partial results (m, sum, accumulators) in the workspace;
// the last worker to arrive merges them in order, so results do not depend on timing.
//
// A warp takes tiles of 16 keys.  Each tile's codes and scales are copied by
// cp.async into the warp's own ring of kStages slots, so that the copies of the
// next tiles are always in flight and no barrier is needed beyond the warp.
// Both products run on the tensor cores:
//   scores   keys on m, query columns on n;
//   outputs  dimensions on m, query columns on n, keys on k.
// Eight columns are more than a few queries fill, so each query takes several.
// int8 keys meet the six bytes of a fixed-point q (46 bits below a power of two
// over its largest: keys whose codes are 0 at a query's large values must not
// inherit their step) in m16n8k32 products, exactly and without any conversion of
// the keys; the last two only where one of the run's is not 0, which fp16 queries
// seldom have (9 x 7 rows fp16: 19.4 us, always 20.7; 32 rows fp32: 15.0 and 14.75.
// The codes are read again for them: held, they made the compiler spill, 21.5).
// e4m3 keys, and the values of both formats, become fp16 exactly and
// meet two fp16 columns, the rounding of q or of a weight and 2^11 times the rest
// (22 bits of its own; q is scaled to 2^14 and weights to 2^7 at their largest, so
// that this holds 2^28 and 2^21 below it).  All columns of a query lie in the same threads, so neither product
// needs a shuffle; `movmatrix` turns the weights into the second one's operand.
// Operand orders are permuted (dimensions of the scores' k, of the outputs' m) so
// that every thread reads 8 or 16 consecutive bytes; the ring's slots are swizzled
// so that those reads have no bank conflicts.
//
// The running reference m is raised, to 2^-7 of the largest weight, only when a
// score exceeds it by 2^15: one vote a tile in place of a maximum over the warp.
constexpr int kAttnWarps = 8;
constexpr float kLead = 7.0f, kLag = 15.0f;   // powers of two of the reference's largest weight and of weights until it is raised
constexpr int kMaxWorkers = 4096;   // counters at the start of the workspace
constexpr float kLoScale = 2048.0f, kLoUnscale = 1.0f / 2048.0f;
constexpr float kNoMax = -3.402823466e38f;    // reference of a column that has seen no key: no finite score is below it

template <int D, int NT>
struct AttnRing {
    static constexpr int kBlocks = D * NT >= 256 ? 1 : 2;   // CTAs per SM; wide column groups need the registers of two
    static constexpr int kStages = (D == 64 ? 6 : 3) * (kBlocks == 1 ? 2 : 1);
    static constexpr int kTileBytes = 32 * D;               // 16 keys' K and V codes
    static constexpr int kLowBytes = 8 * D * NT;            // the last two of six bytes of a run's queries
    template <int FMT, int WPR>
    static constexpr int kSmem = kAttnWarps * kStages * (kTileBytes + 8) + (FMT == G2_KV_I8 ? kAttnWarps / WPR * kLowBytes : 0);
};

struct AttnArgs {
    g2_kv8 c;
    const void *q;
    void *out;
    long long q_stride, out_stride;
    int f16, group;
    float scale_log2e;
    const int *seq_len;
    Rows8 r;
    int unit, ahead;         // keys of a unit; units without keys ahead of a run's
    int workers;             // most workers; fewer where there are fewer units
    unsigned *counters;      // [kMaxWorkers], zero between calls
    float *parts;            // [workers][2][columns * (D + 2)]
};

__device__ __forceinline__ void cp_async4(unsigned dst, const void *src, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ unsigned transpose8x8(unsigned v) {
    unsigned r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float log2_fast(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// v = hi + lo / 2048 of two, each a pair of fp16 (hi in the low half).
__device__ __forceinline__ void split_half2(float v0, float v1, unsigned &s0, unsigned &s1) {
    const __half2 h = __floats2half2_rn(v0, v1);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(fmaf(f.x, -kLoScale, v0 * kLoScale), fmaf(f.y, -kLoScale, v1 * kLoScale));
    const unsigned hb = *reinterpret_cast<const unsigned *>(&h), lb = *reinterpret_cast<const unsigned *>(&l);
    s0 = __byte_perm(hb, lb, 0x5410);
    s1 = __byte_perm(hb, lb, 0x7632);
}

template <int WPR>
__device__ __forceinline__ void group_sync(int group) {
    asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(32 * WPR) : "memory");
}

// Units of sequence s (0 where it has no rows or is out of range).
struct SeqWork {
    int first, n, len, units, col_groups;
    unsigned runs, total;    // total: units of its runs
};
template <int COLS>
__device__ __forceinline__ SeqWork seq_work(const AttnArgs &a, int s) {
    SeqWork w{};
    w.len = a.seq_len[s];   // requested beside the rows' numbers
    const Span sp = seq_rows(a.r, s);
    w.first = sp.first;
    w.n = sp.n;
    if (sp.n <= 0) return w;
    if (w.len < 0 || w.len > (long long)a.r.table_stride * a.c.page_size) {
        bad(a.r);
        w.n = 0;
        return w;
    }
    w.units = max(1, (w.len + a.unit - 1) / a.unit) + a.ahead;   // a row that sees nothing is still written
    w.col_groups = (w.n * a.group + COLS - 1) / COLS;
    w.runs = (unsigned)w.col_groups * a.c.n_kv_head;
    w.total = (unsigned)w.units * w.runs;   // below 2^31 over all sequences: checked on the host
    return w;
}

template <int FMT, int D, int NT, int WPR>
__global__ void __launch_bounds__(kAttnWarps * 32, (AttnRing<D, NT>::kBlocks)) kv8_attention_kernel(AttnArgs a) {
    constexpr int COLS = 4 * NT, KS = D / 16, S = AttnRing<D, NT>::kStages, TILE = AttnRing<D, NT>::kTileBytes, GROUPS = kAttnWarps / WPR;
    constexpr int PART = COLS * (D + 2);
    constexpr bool INT = FMT == G2_KV_I8;
    // slots of a group's first warp that are empty while its queries are staged there
    constexpr int FREE = (NT * KS * 256 + TILE - 1) / TILE;
    static_assert(WPR * PART * 4 <= WPR * S * TILE, "the merge buffer lies in the ring");
    extern __shared__ __align__(128) unsigned char ring[];
    __shared__ unsigned prefix[kAttnWarps * 32];
    __shared__ uint4 warp_sum[kAttnWarps];        // units, runs, longest sequence
    __shared__ int arrived[GROUPS];
    __shared__ SeqWork cached[kAttnWarps * 32];   // of the first sequences
    __shared__ float qfac_s[GROUPS][COLS];        // scores' factor of each query column
    __shared__ int low_s[GROUPS];                 // the run's queries have last bytes that are not 0
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int grp = warp / WPR, wr = warp % WPR, gt = tid - grp * 32 * WPR;
    const int H = a.c.n_kv_head, P = a.c.page_size, n_seq = a.r.n_seq;
    if (gt == 0) low_s[grp] = 0;

    pdl_wait();
    pdl_launch();
    // ---- the units before every `per` sequences
    const int per = (n_seq + kAttnWarps * 32 - 1) / (kAttnWarps * 32);
    unsigned my_units = 0, my_runs = 0, longest = 0;
    bool skipped = false;
    for (int s = tid * per; s < min(n_seq, (tid + 1) * per); ++s) {
        const SeqWork w = seq_work<COLS>(a, s);
        if (per == 1) cached[tid] = w;
        skipped |= w.n < 0;
        my_units += w.total;
        my_runs += w.runs;
        if (w.runs) longest = max(longest, (unsigned)w.len);
    }
    {
        const uint4 x = make_uint4(__reduce_add_sync(0xffffffffu, my_units), __reduce_add_sync(0xffffffffu, my_runs),
                                   __reduce_max_sync(0xffffffffu, longest), 0);
        if (lane == 0) warp_sum[warp] = x;
    }
    if (__syncthreads_or(skipped)) {
        // The host allowed for n_rows rows; where a count was below 0, others may overlap and be more.
        __shared__ unsigned long long units;
        if (tid == 0) units = 0;
        __syncthreads();
        for (int s = tid; s < n_seq; s += kAttnWarps * 32) atomicAdd(&units, (unsigned long long)seq_work<COLS>(a, s).total);
        __syncthreads();
        if (units > 0x7fffffffULL) {
            bad(a.r);
            return;
        }
    }
    uint4 before = make_uint4(0, 0, 0, 0), all = before;
#pragma unroll
    for (int i = 0; i < kAttnWarps; ++i) {
        const uint4 x = warp_sum[i];
        if (i < warp) before = make_uint4(before.x + x.x, before.y + x.y, 0, 0);
        all = make_uint4(all.x + x.x, all.y + x.y, max(all.z, x.z), 0);
    }
    // Whole runs: the longest takes longest / (16 WPR) steps of a worker.  Equal shares are shorter, but partial
    // results and second beginnings cost about kSplitSteps (12 runs of 200 keys: whole 5.2 us, shared 6.5;
    // 12 runs of 1000 keys: whole 8.0, shared 6.7).
    constexpr unsigned kSplitSteps = 4;
    const bool by_run = all.y <= (unsigned)a.workers &&
                        all.z / (16 * WPR) <= (unsigned)((float)all.x * a.unit / (16.0f * WPR * a.workers)) + kSplitSteps;
    const unsigned total = by_run ? all.y : all.x;
    const int unit_keys = by_run ? 0x7fffffff : a.unit, ahead = by_run ? 0 : a.ahead;
    const unsigned mine = by_run ? my_runs : my_units;
    unsigned sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned x = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += x;
    }
    prefix[tid] = (by_run ? before.y : before.x) + sum - mine;
    __syncthreads();
    // A run in p pieces takes units / p steps and then a merge of p: at most kPieces workers a run (one run of
    // 40000 keys over all 296 workers: 25.2 us, 32 pieces: 13.2).
    constexpr unsigned kPieces = 32;
    const unsigned W = min(min((unsigned)a.workers, total), min(all.y, (unsigned)kMaxWorkers) * kPieces);
    const unsigned worker = blockIdx.x * GROUPS + grp;
    if (worker >= W) return;   // whole groups leave; later barriers are the groups' own
    const unsigned share = total / W, extra = total - share * W;   // the first `extra` workers have one unit more
    auto share_begin = [&](unsigned w) { return w * share + min(w, extra); };
    auto worker_of = [&](unsigned unit) {
        const unsigned in_long = extra * (share + 1);
        return unit < in_long ? unit / (share + 1) : extra + (unit - in_long) / share;
    };
    unsigned u = share_begin(worker);
    const unsigned u_end = share_begin(worker + 1);
    auto work_of = [&](int s) {
        SeqWork w = per == 1 ? cached[s] : seq_work<COLS>(a, s);
        if (by_run) {
            w.units = w.runs ? 1 : 0;
            w.total = w.runs;
        }
        return w;
    };

    // ---- the share's first sequence: the last whose units begin at or before u
    int s;
    unsigned seq_begin;
    {
        int n = 0;
#pragma unroll
        for (int i = 0; i < kAttnWarps; ++i) n += __popc(__ballot_sync(0xffffffffu, prefix[i * 32 + lane] <= u));
        s = (n - 1) * per;
        seq_begin = prefix[n - 1];
    }
    SeqWork sw = work_of(s);
    bool first_piece = true;

    unsigned char *slots = ring + warp * S * TILE;
    float *meta = reinterpret_cast<float *>(ring + kAttnWarps * S * TILE) + warp * S * 2;   // K and V scale; -1: no page
    float *merge = reinterpret_cast<float *>(ring + grp * WPR * S * TILE);                  // [WPR][PART]
    uint4 *low = reinterpret_cast<uint4 *>(ring + kAttnWarps * S * (TILE + 8) + grp * AttnRing<D, NT>::kLowBytes);   // [NT][lane][KS / 4]
    const unsigned slots_addr = smem_addr(slots), meta_addr = smem_addr(meta) + lane * 4;   // lanes 0 and 1 bring the scales
    const unsigned char *k_lane = static_cast<const unsigned char *>(a.c.k) + lane * 16, *v_lane = static_cast<const unsigned char *>(a.c.v) + lane * 16;
    const float *scale_lane = lane ? a.c.v_scale : a.c.k_scale;

    // this lane's places in a slot: where it copies to and reads from
    const int crow = lane / (D / 16), ccol = lane % (D / 16);
    const int pv = (crow & 8) | ((crow & 1) << 2) | ((crow >> 1) & 3);   // D = 64: even rows first
    const unsigned k_put = D == 64 ? lane * 16 : crow * 128 + (ccol ^ ((crow & 1) << 2)) * 16;
    const unsigned v_put = 16 * D + (D == 64 ? pv * 64 + (ccol ^ (((pv >> 1) & 1) << 1)) * 16
                                             : crow * 128 + (ccol ^ (((crow >> 1) & 3) << 1)) * 16);

    while (u < u_end) {
        while (u >= seq_begin + sw.total) {   // only past sequences without units or the end of one
            seq_begin += sw.total;
            sw = work_of(++s);
        }
        const unsigned rem = u - seq_begin;
        const int run = (int)(rem / (unsigned)sw.units), unit = (int)rem - run * sw.units;
        const int h = run / sw.col_groups, col0 = run % sw.col_groups * COLS;
        const unsigned run_begin = u - unit, piece_end = min(run_begin + sw.units, u_end);
        // units with keys that are this piece's; the run's first ones may all lie in the next share
        const int unit0 = max(unit - ahead, 0), unit1 = (int)(piece_end - run_begin) - ahead;
        if (unit1 <= 0) break;
        const int cols = min(COLS, sw.n * a.group - col0);
        // key limits of the columns; `lim` of this thread's (column t of each n tile)
        const int lim_first = sw.len - sw.n + col0 / a.group + 1, lim_last = sw.len - sw.n + (col0 + cols - 1) / a.group + 1;
        int lim[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int col = col0 + n * 4 + t;
            lim[n] = n * 4 + t < cols ? sw.len - sw.n + col / a.group + 1 : 0;
        }
        const int kbeg = unit0 * unit_keys;
        const int kend = (int)min((long long)min(sw.len, lim_last), (long long)unit1 * unit_keys);
        const int n_tiles = kend > kbeg ? (kend - kbeg + 15) / 16 : 0;
        const int my_tiles = n_tiles > wr ? (n_tiles - wr + WPR - 1) / WPR : 0;
        const int *table = a.r.table + (long long)s * a.r.table_stride;

        // pages of this warp's tiles, 32 at a time, a window ahead of the copies
        auto load_pages = [&](int base) -> int {
            const int j = base + lane;
            if (j >= my_tiles) return -1;
            const int page = table[(kbeg + (j * WPR + wr) * 16) / P];
            if (page >= 0 && page < a.c.n_pages) return page;
            bad(a.r);
            return -1;
        };
        // the warp's (first) query, ahead of the codes that would delay it
        auto load_query = [&](int c) -> float4 {
            const int col = col0 + c, row = col / a.group, d = lane * 4;
            if (c >= cols || d >= D) return make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            const long long o = (long long)(sw.first + row) * a.q_stride + (long long)(h * a.group + col - row * a.group) * D + d;
            return a.f16 ? load4<__half>(static_cast<const __half *>(a.q) + o) : load4<float>(static_cast<const float *>(a.q) + o);
        };
        float4 x = load_query(wr);
        int pages = load_pages(0), pages_next = my_tiles > 32 ? load_pages(32) : -1;
        int next = 0, key_next = kbeg + wr * 16, put = 0;   // the next tile to copy, its first key, its slot
        auto issue = [&]() {
            if (next < my_tiles) {
                if (next && (next & 31) == 0) {
                    pages = pages_next;
                    pages_next = load_pages(next + 32);
                }
                const int page = __shfl_sync(0xffffffffu, pages, next & 31);
                const unsigned at = (unsigned)max(page, 0) * H + h, row = at * P + (key_next & (P - 1));   // rows fit 32 bits: memory ends first
                const unsigned char *ks = k_lane + (size_t)row * D, *vs = v_lane + (size_t)row * D;
                const unsigned slot = slots_addr + put * TILE, m = meta_addr + put * 8;
                const int rows = page >= 0 ? sw.len - key_next : 0;   // rows from here on are not the sequence's
                if (rows >= 16) {
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) {
                        cp_async16(slot + k_put + i * 512, ks + i * 512, 16);
                        cp_async16(slot + (D == 64 ? v_put : v_put ^ ((i & 1) << 6)) + i * 512, vs + i * 512, 16);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) {
                        const int bytes = crow + i * (512 / D) < rows ? 16 : 0;
                        cp_async16(slot + k_put + i * 512, ks + i * 512, bytes);
                        cp_async16(slot + (D == 64 ? v_put : v_put ^ ((i & 1) << 6)) + i * 512, vs + i * 512, bytes);
                    }
                }
                if (lane < 2) {
                    if (page >= 0) cp_async4(m, scale_lane + at, 4);
                    else asm volatile("st.shared.f32 [%0], %1;" ::"r"(m), "f"(-1.0f) : "memory");
                }
                ++next;
                key_next += 16 * WPR;
                put = put + 1 == S ? 0 : put + 1;
            }
            cp_commit();
        };
#pragma unroll 1
        for (int j = 0; j < S - FREE; ++j) issue();

        // ---- queries, a warp each: into the order of the operands' registers.  Columns 2i and 2i + 1 are of
        // query i; int8 keys have two n tiles, for the upper two and the lower two of the four bytes
        unsigned *qs = reinterpret_cast<unsigned *>(ring + grp * WPR * S * TILE + (S - FREE) * TILE);   // [NT][KS][2][lane]
        unsigned any_low = 0;
        for (int c = wr; c < cols; c += WPR) {
            if (c != wr) x = load_query(c);
            const int d = lane * 4;
            const unsigned peak = __reduce_max_sync(0xffffffffu, max(max(abs_bits(x.x), abs_bits(x.y)), max(abs_bits(x.z), abs_bits(x.w))));
            // a power of two below the largest (2^e <= it < 2^(e + 1)), so that no type's range matters
            const int e = max(INT ? -96 : -112, (int)(peak >> 23) - 127);
            const float down = __uint_as_float((unsigned)(127 + (INT ? 29 : 14) - min(e, 127)) << 23);
            const float up = __uint_as_float((unsigned)(127 + min(e, 127)) << 23) * (INT ? 0x1p-29f : 0x1p-14f);
            if (lane == 0) qfac_s[grp][c] = (peak >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : up) * a.scale_log2e;
            const int k = (d >> 6) * 4 + ((d >> 2) & 3);   // thread (d & 63) >> 4 of a quad has these four dimensions
            unsigned *at = qs + ((c >> 2) * KS * 2) * 32 + (c & 3) * 8 + ((d & 63) >> 4);
            if (d < D) {
                if (INT) {
                    // signed bytes: adding 128 to each of the lower ones carries into the next
                    unsigned z[4];   // 2^15 times what the upper four bytes leave (exact: they have at most the bits of v)
                    auto digits = [&](float v, int i) {
                        const int n = __float2int_rn(v * down);
                        z[i] = ((unsigned)__float2int_rn((v * down - (float)n) * 0x1p15f) + 0x0080u) ^ 0x0080u;
                        return ((unsigned)n + 0x00808080u) ^ 0x00808080u;
                    };
                    const unsigned y0 = digits(x.x, 0), y1 = digits(x.y, 1), y2 = digits(x.z, 2), y3 = digits(x.w, 3);
                    const unsigned z01 = __byte_perm(z[0], z[1], 0x5140), z23 = __byte_perm(z[2], z[3], 0x5140);
                    unsigned *lo = reinterpret_cast<unsigned *>(low) + ((c >> 2) * 32 + (c & 3) * 8 + ((d & 63) >> 4)) * KS + k;
                    any_low |= z01 | z23;
                    lo[0] = __byte_perm(z01, z23, 0x7632);
                    lo[4 * KS] = __byte_perm(z01, z23, 0x5410);
                    const unsigned a01 = __byte_perm(y0, y1, 0x7362), a23 = __byte_perm(y2, y3, 0x7362);   // bytes 2 and 3
                    const unsigned b01 = __byte_perm(y0, y1, 0x5140), b23 = __byte_perm(y2, y3, 0x5140);   // bytes 0 and 1
                    at += ((k >> 1) * 2 + (k & 1)) * 32;
                    at[0] = __byte_perm(a01, a23, 0x7632);
                    at[4] = __byte_perm(a01, a23, 0x5410);
                    at[KS * 32] = __byte_perm(b01, b23, 0x7632);
                    at[KS * 32 + 4] = __byte_perm(b01, b23, 0x5410);
                } else {
                    const __half2 h0 = __floats2half2_rn(x.x * down, x.y * down), h1 = __floats2half2_rn(x.z * down, x.w * down);
                    const float2 f0 = __half22float2(h0), f1 = __half22float2(h1);
                    const __half2 l0 = __floats2half2_rn((x.x * down - f0.x) * kLoScale, (x.y * down - f0.y) * kLoScale);
                    const __half2 l1 = __floats2half2_rn((x.z * down - f1.x) * kLoScale, (x.w * down - f1.y) * kLoScale);
                    at += k * 2 * 32;
                    at[0] = *reinterpret_cast<const unsigned *>(&h0);
                    at[4] = *reinterpret_cast<const unsigned *>(&l0);
                    at[32] = *reinterpret_cast<const unsigned *>(&h1);
                    at[36] = *reinterpret_cast<const unsigned *>(&l1);
                }
            }
        }
        if (INT && any_low) low_s[grp] = 1;
        group_sync<WPR>(grp);
        const bool six = INT && low_s[grp];
        unsigned qf[NT][KS][2];
        float qfac[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {   // columns past the last hold anything: as NaN they never raise a reference
            qfac[n] = n * 4 + t < cols ? qfac_s[grp][n * 4 + t] : __uint_as_float(0x7fc00000u);
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                qf[n][k][0] = qs[((n * KS + k) * 2) * 32 + lane];
                qf[n][k][1] = qs[((n * KS + k) * 2 + 1) * 32 + lane];
            }
        }
        group_sync<WPR>(grp);
        if (gt == 0) low_s[grp] = 0;   // read by all; the next run's queries are two barriers away
#pragma unroll
        for (int j = 1; j < FREE; ++j) issue();

        float acc[NT][KS][4], mref[NT], l[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            mref[n] = kNoMax;
            l[n] = 0.0f;
#pragma unroll
            for (int i = 0; i < KS; ++i)
#pragma unroll
                for (int x = 0; x < 4; ++x) acc[n][i][x] = 0.0f;
        }

        const unsigned char *slot = slots;
        const float *mt = meta;
        for (int j = 0, key0 = kbeg + wr * 16; j < my_tiles; ++j, key0 += 16 * WPR) {
            cp_wait<S - 2>();
            __syncwarp();
            issue();
            // ---- scores
            float sc[NT][2];   // of keys g and g + 8
            if constexpr (INT) {
                auto pair = [](const int (&v)[4], int j) { return (float)(v[2 * j] * 256 + v[2 * j + 1]); };
                // keys g and g + 8 of the tile, 32 dimensions in each product
                auto keys = [&](int b, unsigned (&f0)[4], unsigned (&f1)[4]) {
                    const int c = D == 64 ? t : (b * 4 + t) ^ ((g & 1) << 2);
                    const uint4 r0 = *reinterpret_cast<const uint4 *>(slot + g * D + c * 16);
                    const uint4 r1 = *reinterpret_cast<const uint4 *>(slot + (g + 8) * D + c * 16);
                    f0[0] = r0.x, f0[1] = r1.x, f0[2] = r0.y, f0[3] = r1.y;
                    f1[0] = r0.z, f1[1] = r1.z, f1[2] = r0.w, f1[3] = r1.w;
                };
#pragma unroll
                for (int n = 0; n < NT; ++n) sc[n][0] = sc[n][1] = 0.0f;
                if (six) {   // the last two bytes
                    int s[NT][4];
#pragma unroll
                    for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0;
#pragma unroll
                    for (int b = 0; b < D / 64; ++b) {
                        unsigned f0[4], f1[4];
                        keys(b, f0, f1);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            const uint4 lo = low[(n * 32 + lane) * (KS / 4) + b];
                            mma16832(s[n], f0, lo.x, lo.y);
                            mma16832(s[n], f1, lo.z, lo.w);
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        sc[n][0] = pair(s[n], 0) * 0x1p-15f;
                        sc[n][1] = pair(s[n], 1) * 0x1p-15f;
                    }
                }
                int s[NT][2][4];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 2; ++i) s[n][i][0] = s[n][i][1] = s[n][i][2] = s[n][i][3] = 0;
#pragma unroll
                for (int b = 0; b < D / 64; ++b) {
                    unsigned f0[4], f1[4];
                    keys(b, f0, f1);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            mma16832(s[n][i], f0, qf[n][i * (KS / 2) + b * 2][0], qf[n][i * (KS / 2) + b * 2][1]);
                            mma16832(s[n][i], f1, qf[n][i * (KS / 2) + b * 2 + 1][0], qf[n][i * (KS / 2) + b * 2 + 1][1]);
                        }
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    sc[n][0] = fmaf(pair(s[n][0], 0), 65536.0f, pair(s[n][1], 0) + sc[n][0]);
                    sc[n][1] = fmaf(pair(s[n][0], 1), 65536.0f, pair(s[n][1], 1) + sc[n][1]);
                }
            } else {
                float s[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
#pragma unroll
                for (int b = 0; b < D / 64; ++b) {
                    const int c = D == 64 ? t : (b * 4 + t) ^ ((g & 1) << 2);
                    const uint4 r0 = *reinterpret_cast<const uint4 *>(slot + g * D + c * 16);
                    const uint4 r1 = *reinterpret_cast<const uint4 *>(slot + (g + 8) * D + c * 16);
                    const unsigned w0[4] = {r0.x, r0.y, r0.z, r0.w}, w1[4] = {r1.x, r1.y, r1.z, r1.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        unsigned f[4];
                        codes_to_half<FMT>(w0[i], f[0], f[2]);
                        codes_to_half<FMT>(w1[i], f[1], f[3]);
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma16816(s[n], f, qf[n][b * 4 + i][0], qf[n][b * 4 + i][1]);
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    sc[n][0] = fmaf(s[n][1], kLoUnscale, s[n][0]);
                    sc[n][1] = fmaf(s[n][3], kLoUnscale, s[n][2]);
                }
            }
            // ---- weights
            const float2 scales = *reinterpret_cast<const float2 *>(mt);
            const bool there = !(scales.y < 0.0f);                              // a NaN scale is there
            const float vs = scales.y < kScaleFloor ? kScaleFloor : scales.y;   // and stays NaN
            const float lvs = there ? log2_fast(vs) : -INFINITY, rvs = rcp_fast(vs);
            const bool all = key0 + 16 <= lim_first;
            float w[NT][2];
            bool raise = false;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float f = there ? scales.x * qfac[n] : 0.0f;
                w[n][0] = fmaf(sc[n][0], f, lvs);
                w[n][1] = fmaf(sc[n][1], f, lvs);
                if (!all) {
                    if (key0 + g >= lim[n]) w[n][0] = -INFINITY;
                    if (key0 + g + 8 >= lim[n]) w[n][1] = -INFINITY;
                }
                raise |= fmaxf(w[n][0], w[n][1]) > mref[n] + kLag;
            }
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float m = fmaxf(fmaxf(w[n][0], w[n][1]) - kLead, mref[n]);
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                    const float fix = exp2_fast(mref[n] - m);
                    mref[n] = m;
                    l[n] *= fix;
#pragma unroll
                    for (int i = 0; i < KS; ++i)
#pragma unroll
                        for (int x = 0; x < 4; ++x) acc[n][i][x] *= fix;
                }
            }
            unsigned pb[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float p0 = exp2_fast(w[n][0] - mref[n]), p1 = exp2_fast(w[n][1] - mref[n]);
                if (p0 + p1 != 0.0f) l[n] = fmaf(p0 + p1, rvs, l[n]);   // a NaN scale reaches only columns that see it
                unsigned s0, s1;
                split_half2(p0, p1, s0, s1);
                pb[n][0] = transpose8x8(s0);
                pb[n][1] = transpose8x8(s1);
            }
            // ---- outputs: keys 2t, 2t + 1, 2t + 8, 2t + 9 of this thread's D / 8 dimensions
            const unsigned char *vslot = slot + 16 * D;
            unsigned v[4][D / 32];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int row = 2 * t + (x & 1) + (x >> 1) * 8;
                if (D == 64) {
                    const int pr = (row & 8) | ((row & 1) << 2) | ((row >> 1) & 3);
                    const uint2 r = *reinterpret_cast<const uint2 *>(vslot + pr * 64 + ((g >> 1) ^ (((pr >> 1) & 1) << 1)) * 16 + (g & 1) * 8);
                    v[x][0] = r.x;
                    v[x][1] = r.y;
                } else {
                    const uint4 r = *reinterpret_cast<const uint4 *>(vslot + row * 128 + (g ^ (((row >> 1) & 3) << 1)) * 16);
                    const unsigned all4[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
                    for (int y = 0; y < D / 32; ++y) v[x][y] = all4[y];
                }
            }
#pragma unroll
            for (int i = 0; i < KS; ++i) {   // dimensions 2i and 2i + 1 of the thread's
                const unsigned sel = (i & 1) ? 0x7362 : 0x5140;
                unsigned f[4];
                codes_to_half<FMT>(__byte_perm(v[0][i / 2], v[1][i / 2], sel), f[0], f[1]);
                codes_to_half<FMT>(__byte_perm(v[2][i / 2], v[3][i / 2], sel), f[2], f[3]);
#pragma unroll
                for (int n = 0; n < NT; ++n) mma16816(acc[n][i], f, pb[n][0], pb[n][1]);
            }
            slot = slot + TILE == slots + S * TILE ? slots : slot + TILE;
            mt = mt + 2 == meta + S * 2 ? meta : mt + 2;
        }
        cp_wait<0>();

        // ---- the warps' results of this piece, into the ring's memory
        group_sync<WPR>(grp);
        float *mw = merge + wr * PART;   // [COLS][D] sums, [COLS] references, [COLS] weights
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            l[n] += __shfl_xor_sync(0xffffffffu, l[n], 4);
            l[n] += __shfl_xor_sync(0xffffffffu, l[n], 8);
            l[n] += __shfl_xor_sync(0xffffffffu, l[n], 16);
            const int c = n * 4 + t;
            if (g == 0) {
                mw[COLS * D + c] = mref[n];
                mw[COLS * (D + 1) + c] = l[n];
            }
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                float2 o;
                o.x = fmaf(acc[n][i][1], kLoUnscale, acc[n][i][0]);
                o.y = fmaf(acc[n][i][3], kLoUnscale, acc[n][i][2]);
                *reinterpret_cast<float2 *>(mw + c * D + g * (D / 8) + 2 * i) = o;
            }
        }
        group_sync<WPR>(grp);

        const bool whole = unit0 == 0 && unit1 == sw.units - ahead;
        float *part = a.parts + ((size_t)worker * 2 + (first_piece ? 0 : 1)) * PART;
        auto store = [&](int i, float v) {
            const int c = i / D, d = i % D, col = col0 + c, row = col / a.group;
            const long long o = (long long)(sw.first + row) * a.out_stride + (long long)(h * a.group + col - row * a.group) * D + d;
            if (a.f16) static_cast<__half *>(a.out)[o] = __float2half_rn(v);
            else static_cast<float *>(a.out)[o] = v;
        };
        for (int i = gt; i < cols * D; i += 32 * WPR) {
            const int c = i / D, d = i % D;
            float m = kNoMax, sum_w = 0.0f, sum_o = 0.0f;
#pragma unroll
            for (int x = 0; x < WPR; ++x) m = fmaxf(m, merge[x * PART + COLS * D + c]);
#pragma unroll
            for (int x = 0; x < WPR; ++x) {
                const float fix = exp2_fast(merge[x * PART + COLS * D + c] - m);
                sum_w = fmaf(merge[x * PART + COLS * (D + 1) + c], fix, sum_w);
                sum_o = fmaf(merge[x * PART + c * D + d], fix, sum_o);
            }
            if (whole) {
                store(i, sum_w == 0.0f ? 0.0f : sum_o / sum_w);
            } else {
                part[i] = sum_o;
                if (d == 0) {
                    part[COLS * D + c] = m;
                    part[COLS * (D + 1) + c] = sum_w;
                }
            }
        }
        if (!whole) {
            const unsigned w0 = worker_of(run_begin + ahead), w1 = worker_of(run_begin + sw.units - 1);
            group_sync<WPR>(grp);
            if (gt == 0) {   // releases the group's results and acquires the others'
                unsigned seen;
                asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(seen) : "l"(a.counters + w0) : "memory");
                arrived[grp] = (int)seen;
            }
            group_sync<WPR>(grp);
            if (arrived[grp] == (int)(w1 - w0)) {   // every other piece is there
                if (gt == 0) a.counters[w0] = 0;
                // piece of worker x: its first one, or, where the run begins inside the share, its last
                const float *piece0 = a.parts + ((size_t)w0 * 2 + (share_begin(w0) < run_begin ? 1 : 0)) * PART;
                const float *pieces = a.parts + (size_t)w0 * 2 * PART;
                const int n = (int)(w1 - w0) + 1;
                constexpr int TH = 32 * WPR, PER = COLS * D > TH ? 2 : 1;   // outputs of a thread taken together
                for (int i0 = gt; i0 < cols * D; i0 += PER * TH) {
                    float m[PER], sum_w[PER], sum_o[PER];
#pragma unroll
                    for (int z = 0; z < PER; ++z) {
                        m[z] = kNoMax;
                        sum_w[z] = sum_o[z] = 0.0f;
                    }
                    for (int x = 0; x < n; x += 8) {   // the loads of eight pieces at a time; summed in order
                        float pm[PER][8], pw[PER][8], po[PER][8];
#pragma unroll
                        for (int y = 0; y < 8; ++y) {
                            const float *p = x + y == 0 ? piece0 : pieces + (size_t)(x + y) * 2 * PART;
#pragma unroll
                            for (int z = 0; z < PER; ++z) {
                                const int i = i0 + z * TH, c = i / D;
                                const bool there = x + y < n && i < cols * D;
                                pm[z][y] = there ? __ldcg(p + COLS * D + c) : kNoMax;
                                pw[z][y] = there ? __ldcg(p + COLS * (D + 1) + c) : 0.0f;
                                po[z][y] = there ? __ldcg(p + i) : 0.0f;
                            }
                        }
#pragma unroll
                        for (int z = 0; z < PER; ++z) {
                            float nm = m[z];
#pragma unroll
                            for (int y = 0; y < 8; ++y) nm = fmaxf(nm, pm[z][y]);
                            const float f = exp2_fast(m[z] - nm);
                            m[z] = nm;
                            sum_w[z] *= f;
                            sum_o[z] *= f;
#pragma unroll
                            for (int y = 0; y < 8; ++y) {
                                const float fix = exp2_fast(pm[z][y] - nm);
                                sum_w[z] = fmaf(pw[z][y], fix, sum_w[z]);
                                sum_o[z] = fmaf(po[z][y], fix, sum_o[z]);
                            }
                        }
                    }
#pragma unroll
                    for (int z = 0; z < PER; ++z)
                        if (i0 + z * TH < cols * D) store(i0 + z * TH, sum_w[z] == 0.0f ? 0.0f : sum_o[z] / sum_w[z]);
                }
            }
        }
        group_sync<WPR>(grp);   // the merge buffer is the next piece's ring
        first_piece = false;
        u = piece_end;
    }
}

// Query columns a warp works on together, and how the work is cut.
struct AttnPlan {
    int nt, wpr, unit, ahead, workers;
    size_t part_floats;
};
AttnPlan attn_plan(const g2_kv8 &c, int n_head, int n_seq, int max_q, int sms) {
    AttnPlan p;
    const long long cols = (long long)max_q * (n_head / c.n_kv_head);
    p.nt = cols <= 4 ? 1 : cols <= 8 || c.head_dim == 128 ? 2 : 4;
    const long long runs = (long long)n_seq * c.n_kv_head * ((cols + 4 * p.nt - 1) / (4 * p.nt));
    // Few runs: eight warps share one, as each crosses many workers.  Many: pairs of warps, so that the
    // beginnings and ends of runs overlap (32 x 16 runs of up to 1024 keys: 13.9 us, eight warps 16.6;
    // 4 x 8 runs of up to 65536: 57.6, pairs 76).  `ahead` evens the workers' times where runs are short
    // (9 x 25 runs of up to 2021 keys: 18.4, without it 24.7).
    const bool many = runs >= 2LL * sms;
    p.wpr = many ? 2 : 8;
    p.unit = many ? 64 : 128;
    p.ahead = many ? 2 : 3;
    p.workers = sms * (c.head_dim * p.nt >= 256 ? 1 : 2) * (kAttnWarps / p.wpr);
    if (p.workers > kMaxWorkers) p.workers = kMaxWorkers;
    p.part_floats = (size_t)p.workers * 2 * 4 * p.nt * (c.head_dim + 2);
    return p;
}

template <int FMT, int D, int NT, int WPR>
int launch_attn(const AttnArgs &a, cudaStream_t st) {
    auto kernel = kv8_attention_kernel<FMT, D, NT, WPR>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (AttnRing<D, NT>::template kSmem<FMT, WPR>)) != cudaSuccess)
        return arg_error(G2_ERR_CUDA, "g2k_kv8_attention", cudaGetErrorString(cudaGetLastError()));
    const int per_cta = kAttnWarps / WPR;
    return launch_status("g2k_kv8_attention", launch_pdl(kernel, dim3((a.workers + per_cta - 1) / per_cta), dim3(kAttnWarps * 32),
                                                         (AttnRing<D, NT>::template kSmem<FMT, WPR>), st, a));
}

template <int FMT, int D, int NT>
int launch_attn(const AttnArgs &a, int wpr, cudaStream_t st) {
    return wpr == 2 ? launch_attn<FMT, D, NT, 2>(a, st) : launch_attn<FMT, D, NT, 8>(a, st);
}

template <int FMT>
int launch_attn(const AttnArgs &a, const AttnPlan &p, cudaStream_t st) {
    if (a.c.head_dim == 64)
        return p.nt == 1 ? launch_attn<FMT, 64, 1>(a, p.wpr, st)
             : p.nt == 2 ? launch_attn<FMT, 64, 2>(a, p.wpr, st) : launch_attn<FMT, 64, 4>(a, p.wpr, st);
    return p.nt == 1 ? launch_attn<FMT, 128, 1>(a, p.wpr, st) : launch_attn<FMT, 128, 2>(a, p.wpr, st);
}

// Positions of a table row: the attention counts up to a unit of keys past the last in 32 bits.
constexpr long long kMaxPositions = 0x7fffff00LL;

// ---- argument checks ----------------------------------------------------------------
int check_cache(const char *who, const g2_kv8 *c) {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) return arg_error(G2_ERR_ARG, who, "null cache or cache array");
    if (c->format != G2_KV_I8 && c->format != G2_KV_E4M3) return arg_error(G2_ERR_ARG, who, "bad cache format");
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
        return arg_error(G2_ERR_ARG, who, "page_size must be 16, 32, 64 or 128");
    if (c->head_dim != 64 && c->head_dim != 128) return arg_error(G2_ERR_ARG, who, "head_dim must be 64 or 128");
    if (c->n_pages < 1 || c->n_kv_head < 1 || c->n_kv_head > 32767)   // append's grid has a row for each head's K and V
        return arg_error(G2_ERR_RANGE, who, "need n_pages >= 1 and 1 <= n_kv_head <= 32767");
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4))
        return arg_error(G2_ERR_ARG, who, "codes must be 16-byte aligned, scales 4-byte");
    return G2_OK;
}

// Everything but the pointers' memory; strides become elements.
int check_rows(const char *who, const g2_kv8 *c, int heads, const void *a, const void *b, int dtype, long long *sa,
               long long *sb, const Rows8 &r, const int *per_seq) {
    if (!a || !b || !r.table || !per_seq) return arg_error(G2_ERR_ARG, who, "null argument");
    if (dtype != G2_F32 && dtype != G2_F16) return arg_error(G2_ERR_ARG, who, "bad dtype");
    if (r.n_rows < 0 || r.n_seq < 0 || r.max_q < 1 || r.table_stride < 1)
        return arg_error(G2_ERR_RANGE, who, "need n_rows >= 0, n_seq >= 0, max_q >= 1 and table_stride >= 1");
    if (!r.q_start && (r.max_q != 1 || r.n_rows != r.n_seq))
        return arg_error(G2_ERR_RANGE, who, "without q_start n_rows is n_seq and max_q is 1");
    if ((long long)r.table_stride * c->page_size > kMaxPositions)
        return arg_error(G2_ERR_RANGE, who, "a table row holds more than 2^31 - 256 positions");
    const int es = dtype == G2_F32 ? 4 : 2;
    for (long long *s : {sa, sb}) {
        if (!s) continue;
        if (*s == 0) *s = (long long)heads * c->head_dim;
        if (*s < (long long)heads * c->head_dim) return arg_error(G2_ERR_RANGE, who, "a row stride is less than a row");
        if (*s * es % 16) return arg_error(G2_ERR_ARG, who, "row strides must be multiples of 16 bytes");
    }
    if (!aligned(a, 16) || !aligned(b, 16)) return arg_error(G2_ERR_ARG, who, "rows must be 16-byte aligned");
    if (!aligned(r.table, 4) || !aligned(r.q_start, 4) || !aligned(per_seq, 4) || !aligned(r.status, 4))
        return arg_error(G2_ERR_ARG, who, "an int array is not 4-byte aligned");
    return G2_OK;
}

template <typename T, int FMT>
cudaError_t launch_append(const g2_kv8 &c, const void *k, const void *v, long long stride, const int *pos, const Rows8 &r,
                   cudaStream_t st) {
    const T *kt = static_cast<const T *>(k), *vt = static_cast<const T *>(v);
    if (r.max_q == 1) {
        const dim3 grid(r.n_seq, (2 * c.n_kv_head + 7) / 8);
        return c.head_dim == 64 ? launch_pdl(kv8_append_token_kernel<T, FMT, 64>, grid, dim3(256), 0, st, c, kt, vt, stride, pos, r)
                                : launch_pdl(kv8_append_token_kernel<T, FMT, 128>, grid, dim3(256), 0, st, c, kt, vt, stride, pos, r);
    }
    const int per = (int)(((long long)c.page_size + r.max_q - 2) / c.page_size) + 1;   // blocks that max_q rows can touch
    const int vpt = c.page_size * c.head_dim / (4 * kAppendThreads), tiles = std::max(1, kAppendVecs / vpt);
    const dim3 grid((unsigned)per * r.n_seq, (2 * c.n_kv_head + tiles - 1) / tiles);
    auto launch = [&](auto kernel) { return launch_pdl(kernel, grid, dim3(kAppendThreads), 0, st, c, kt, vt, stride, pos, r, per); };
    if (c.head_dim == 64) {
        switch (vpt) {
            case 1: return launch(kv8_append_kernel<T, FMT, 64, 1>);
            case 2: return launch(kv8_append_kernel<T, FMT, 64, 2>);
            case 4: return launch(kv8_append_kernel<T, FMT, 64, 4>);
            default: return launch(kv8_append_kernel<T, FMT, 64, 8>);
        }
    } else {
        switch (vpt) {
            case 2: return launch(kv8_append_kernel<T, FMT, 128, 2>);
            case 4: return launch(kv8_append_kernel<T, FMT, 128, 4>);
            case 8: return launch(kv8_append_kernel<T, FMT, 128, 8>);
            default: return launch(kv8_append_kernel<T, FMT, 128, 16>);
        }
    }
}

template <typename T, int FMT>
cudaError_t launch_gather(const g2_kv8 &c, void *k, void *v, long long stride, const int *pos, const Rows8 &r, cudaStream_t st) {
    const int per = (int)(((long long)r.max_q + kGatherRows - 2) / kGatherRows) + 1;   // chunks that max_q rows can touch
    const dim3 grid((unsigned)per * r.n_seq, (c.n_kv_head * c.head_dim / 2 + 255) / 256);
    return launch_pdl(kv8_gather_kernel<T, FMT>, grid, dim3(256), 0, st, c, static_cast<T *>(k), static_cast<T *>(v), stride, pos, r, per);
}

// A sequence has no more rows than there are: a larger bound only makes larger grids.
int bound_rows(int max_q, int n_rows) { return std::min(max_q, std::max(n_rows, 1)); }

// dtype and format to template arguments
#define G2_KV8_DISPATCH(fn, ...)                                                                                       \
    (dtype == G2_F32 ? (cache->format == G2_KV_I8 ? fn<float, G2_KV_I8>(__VA_ARGS__) : fn<float, G2_KV_E4M3>(__VA_ARGS__)) \
                     : (cache->format == G2_KV_I8 ? fn<__half, G2_KV_I8>(__VA_ARGS__) : fn<__half, G2_KV_E4M3>(__VA_ARGS__)))

}  // namespace

}  // namespace g2

using namespace g2;

extern "C" int g2k_kv8_append(const g2_kv8 *cache, const void *k, const void *v, int dtype, long long row_stride, int n_rows,
                              int n_seq, const int *q_start, const int *pos, int max_q, const int *table, int table_stride,
                              int *status, void *stream) {
    const char *who = "g2k_kv8_append";
    int rc;
    if ((rc = check_cache(who, cache))) return rc;
    Rows8 r{n_rows, n_seq, max_q, q_start, table, table_stride, status};
    if ((rc = check_rows(who, cache, cache->n_kv_head, k, v, dtype, &row_stride, nullptr, r, pos))) return rc;
    r.max_q = bound_rows(max_q, n_rows);
    if (((long long)r.max_q / cache->page_size + 3) * n_seq > 0x7fffffffLL) return arg_error(G2_ERR_RANGE, who, "too many blocks");
    if (n_rows == 0 || n_seq == 0) return G2_OK;
    if ((rc = check_device_ptrs(who, {cache->k, cache->v, cache->k_scale, cache->v_scale, k, v, q_start, pos, table, status})))
        return rc;
    return launch_status(who, G2_KV8_DISPATCH(launch_append, *cache, k, v, row_stride, pos, r, (cudaStream_t)stream));
}

extern "C" int g2k_kv8_gather(const g2_kv8 *cache, void *k_out, void *v_out, int dtype, long long row_stride, int n_rows,
                              int n_seq, const int *q_start, const int *pos, int max_q, const int *table, int table_stride,
                              int *status, void *stream) {
    const char *who = "g2k_kv8_gather";
    int rc;
    if ((rc = check_cache(who, cache))) return rc;
    Rows8 r{n_rows, n_seq, max_q, q_start, table, table_stride, status};
    if ((rc = check_rows(who, cache, cache->n_kv_head, k_out, v_out, dtype, &row_stride, nullptr, r, pos))) return rc;
    r.max_q = bound_rows(max_q, n_rows);
    if (((long long)r.max_q / kGatherRows + 3) * n_seq > 0x7fffffffLL) return arg_error(G2_ERR_RANGE, who, "too many rows");
    if (n_rows == 0 || n_seq == 0) return G2_OK;
    if ((rc = check_device_ptrs(who, {cache->k, cache->v, cache->k_scale, cache->v_scale, k_out, v_out, q_start, pos, table, status})))
        return rc;
    return launch_status(who, G2_KV8_DISPATCH(launch_gather, *cache, k_out, v_out, row_stride, pos, r, (cudaStream_t)stream));
}

// [counters | partial results], each 256-byte aligned; the counters' place does not depend on the call's sizes
extern "C" size_t g2k_kv8_attention_workspace(const g2_kv8 *cache, int n_head, int n_seq, int max_q) {
    if (!cache || n_head < 1 || n_seq < 0 || max_q < 1 || cache->n_kv_head < 1 || n_head % cache->n_kv_head) return 0;
    return kMaxWorkers * 4 + attn_plan(*cache, n_head, n_seq, max_q, sm_count()).part_floats * 4;
}

extern "C" int g2k_kv8_attention(const g2_kv8 *cache, const void *q, long long q_stride, void *out, long long out_stride,
                                 int dtype, int n_head, float scale, int n_rows, int n_seq, const int *q_start,
                                 const int *seq_len, int max_q, const int *table, int table_stride, void *workspace,
                                 size_t workspace_bytes, int *status, void *stream) {
    const char *who = "g2k_kv8_attention";
    int rc;
    if ((rc = check_cache(who, cache))) return rc;
    if (n_head < 1 || n_head % cache->n_kv_head || n_head > 65535)
        return arg_error(G2_ERR_RANGE, who, "n_head must be a multiple of n_kv_head, at most 65535");
    constexpr float kLog2e = 1.4426950408889634f;
    if (!(scale > 0.0f) || !std::isfinite(scale * kLog2e)) return arg_error(G2_ERR_ARG, who, "scale must be positive and at most 2.3e38");
    Rows8 r{n_rows, n_seq, max_q, q_start, table, table_stride, status};
    if ((rc = check_rows(who, cache, n_head, q, out, dtype, &q_stride, &out_stride, r, seq_len))) return rc;
    r.max_q = bound_rows(max_q, n_rows);
    if ((long long)r.max_q * n_seq > 0x7fffffffLL) return arg_error(G2_ERR_RANGE, who, "too many rows");
    {   // the kernel counts units in 32 bits: those of the longest sequences, for each group of query columns (the last
        // of a sequence may be part full)
        const AttnPlan p = attn_plan(*cache, n_head, n_seq, r.max_q, 1);
        const double columns = (double)std::min((long long)r.max_q * n_seq, (long long)n_rows) * (n_head / cache->n_kv_head);
        const double units = ((double)table_stride * cache->page_size / p.unit + 1 + p.ahead) * cache->n_kv_head *
                             (columns / (4 * p.nt) + std::min(n_seq, n_rows));
        if (units > 2147483647.0) return arg_error(G2_ERR_RANGE, who, "too much work for one call");
    }
    if (!workspace || !aligned(workspace, 256)) return arg_error(G2_ERR_ARG, who, "workspace not 256-byte aligned");
    if (workspace_bytes < g2k_kv8_attention_workspace(cache, n_head, n_seq, max_q))
        return arg_error(G2_ERR_ARG, who, "workspace too small");
    if (n_rows == 0 || n_seq == 0) return G2_OK;
    if ((rc = check_device_ptrs(who, {cache->k, cache->v, cache->k_scale, cache->v_scale, q, out, q_start, seq_len, table,
                                      workspace, status})))
        return rc;
    const AttnPlan p = attn_plan(*cache, n_head, n_seq, r.max_q, sm_count());   // needs no more workspace than max_q's plan
    const AttnArgs a{*cache, q, out, q_stride, out_stride, dtype == G2_F16, n_head / cache->n_kv_head,
                     scale * kLog2e, seq_len, r, p.unit, p.ahead, p.workers, static_cast<unsigned *>(workspace),
                     static_cast<float *>(workspace) + kMaxWorkers};
    return cache->format == G2_KV_I8 ? launch_attn<G2_KV_I8>(a, p, (cudaStream_t)stream)
                                     : launch_attn<G2_KV_E4M3>(a, p, (cudaStream_t)stream);
}
