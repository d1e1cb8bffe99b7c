// g2_q4.cu -- weights in 4 bits: packing (g2k_q4_pack), reading back
// (g2k_q4_unpack) and the matrix-vector product on them (g2k_matvec_q4).
//
// W [K][N] is cut into groups of `group` rows of a column.  A group's scale is
// s = bf16(max|w| / 7) and its codes c = w / s rounded, in -7..7, so that
//   y[m][n] = sum_groups s[g][n] * sum_{k in g} x'[m][k] c[k][n].
//
// Packed layout, for tiles of 16 columns (features) and chunks of 64 rows, in the
// order in which the product reads them:
//   [tile][chunk] { codes [lane 0..31][4 words], scales [1, or 2 for groups of 32][8][2] bf16 }
// A scale pair is that of features g and g + 8; a group of 128 rows has its scale
// in both of its chunks (3% more bytes, and a chunk needs nothing but itself).
// Word s of lane (g = lane / 4, t = lane % 4) holds features g (upper nibbles) and
// g + 8 (lower nibbles) at rows 64 chunk + 32 (s / 2) + 8 t + 4 (s % 2) + {0, 2, 1, 3}
// of its bytes 0..3, as two's complement.  Such a word is a thread's part of the A
// operand of one 16 x 8 x 16 product of fp16 (registers: upper and lower nibbles of
// bytes 0 and 2, of bytes 1 and 3), or half of it of one 16 x 8 x 32 product of int8
// (registers: upper nibbles, lower nibbles); the k index is a permutation of the rows,
// under which the x of a lane are consecutive.  Rows past K and columns past N, up
// to a multiple of 32, hold code 0.
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

#include "g2_args.h"
#include "g2_device.cuh"
#include "g2_mma.cuh"

namespace g2 {

namespace {

constexpr int kTile = 16, kChunk = 64;

struct Q4Shape {
    int N, K, group;
    int tiles, chunks;
    int per_chunk;       // scale groups of a chunk
    int chunk_bytes;
    __host__ __device__ Q4Shape(int N_, int K_, int group_) : N(N_), K(K_), group(group_) {
        tiles = (N + 2 * kTile - 1) / (2 * kTile) * 2;   // in pairs
        chunks = (K + kChunk - 1) / kChunk;
        per_chunk = group == 32 ? 2 : 1;
        chunk_bytes = 512 + 32 * per_chunk;
    }
    size_t bytes() const { return (size_t)tiles * chunks * chunk_bytes; }
    __device__ size_t at(int tile, int chunk) const { return ((size_t)tile * chunks + chunk) * chunk_bytes; }
};

// w / s rounded to the nearest integer, ties to even, from the exact quotient:
// q is within one of it, and the remainder w - q s is exact in one fma.
__device__ __forceinline__ int round_quotient(float w, float s) {
    float q = rintf(__fdiv_rn(w, s));
    const float r = __fmaf_rn(-q, s, w), h = 0.5f * s;
    if (r > h || (r == h && ((int)q & 1))) q += 1.0f;
    if (r < -h || (r == -h && ((int)q & 1))) q -= 1.0f;
    return (int)q;
}

// One CTA per (tile, group): the group's largest magnitudes, then its codes.
constexpr int kPackThreads = 128;

template <typename T>
__global__ void __launch_bounds__(kPackThreads) q4_pack_kernel(const T *W, int transposed, unsigned char *packed,
                                                               Q4Shape sh) {
    __shared__ unsigned peak[kTile];
    __shared__ float step[kTile];
    __shared__ unsigned char code[128][kTile];
    const int tile = blockIdx.x, grp = blockIdx.y, t = threadIdx.x;
    const int k0 = grp * sh.group, n0 = tile * kTile;
    if (t < kTile) peak[t] = 0;
    __syncthreads();
    // consecutive threads follow the array's rows
    auto at = [&](int i, int &f, int &k) {
        if (transposed) {
            k = i % sh.group;
            f = i / sh.group;
        } else {
            f = i % kTile;
            k = i / kTile;
        }
    };
    auto load = [&](int f, int k) -> float {
        if (n0 + f >= sh.N || k0 + k >= sh.K) return 0.0f;
        return tof(transposed ? W[(size_t)(n0 + f) * sh.K + k0 + k] : W[(size_t)(k0 + k) * sh.N + n0 + f]);
    };
    for (int i = t; i < sh.group * kTile; i += kPackThreads) {
        int f, k;
        at(i, f, k);
        atomicMax(&peak[f], __float_as_uint(fabsf(load(f, k))));   // as integers: NaN above infinity above finite
    }
    __syncthreads();
    if (t < kTile) {
        const __nv_bfloat16 s = __float2bfloat16_rn(__fdiv_rn(__uint_as_float(peak[t]), 7.0f));
        step[t] = __bfloat162float(s);
        const __nv_bfloat16 v = peak[t] >= 0x7f800000u ? __ushort_as_bfloat16(0x7fc0) : s;
        for (int c = k0 / kChunk; c * kChunk < k0 + sh.group && c < sh.chunks; ++c) {
            auto *o = reinterpret_cast<__nv_bfloat16 *>(packed + sh.at(tile, c) + 512 + (k0 % kChunk) / 32 * 32);
            o[(t & 7) * 2 + (t >> 3)] = v;
        }
    }
    __syncthreads();
    for (int i = t; i < sh.group * kTile; i += kPackThreads) {
        int f, k;
        at(i, f, k);
        const float s = step[f];
        int c = 0;
        if (s > 0.0f && peak[f] < 0x7f800000u) c = max(-7, min(7, round_quotient(load(f, k), s)));
        code[k][f] = (unsigned char)(c & 15);
    }
    __syncthreads();
    // 32 lanes per 16 rows
    for (int i = t; i < sh.group * 2; i += kPackThreads) {
        const int lane = i & 31, step16 = i >> 5, kk = k0 + step16 * 16;
        const int chunk = kk / kChunk, s = (kk % kChunk) / 16;
        if (chunk >= sh.chunks) continue;
        const int g = lane >> 2, r = chunk * kChunk + 32 * (s >> 1) + 8 * (lane & 3) + 4 * (s & 1) - k0;
        unsigned w = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int shift = 16 * (j & 1) + 8 * (j >> 1);
            w |= (unsigned)(code[r + j][g] << 4 | code[r + j][g + 8]) << shift;
        }
        reinterpret_cast<unsigned *>(packed + sh.at(tile, chunk))[lane * 4 + s] = w;
    }
}

__global__ void __launch_bounds__(256) q4_unpack_kernel(const unsigned char *packed, float *W, Q4Shape sh) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long long)sh.K * sh.N) return;
    const int k = (int)(i / sh.N), n = (int)(i % sh.N);
    const int f = n % kTile, kc = k % kChunk, r = kc & 3;
    const int lane = (f & 7) * 4 + ((kc >> 3) & 3), s = (kc >> 5) * 2 + ((kc >> 2) & 1);
    const unsigned char *chunk = packed + sh.at(n / kTile, k / kChunk);
    const unsigned w = reinterpret_cast<const unsigned *>(chunk)[lane * 4 + s];
    const int shift = 16 * (r & 1) + 8 * (r >> 1) + (f < 8 ? 4 : 0);
    const auto *scale = reinterpret_cast<const __nv_bfloat16 *>(chunk + 512 + (sh.per_chunk == 2 ? kc / 32 * 32 : 0));
    W[i] = (float)((int)(w << (28 - shift)) >> 28) * __bfloat162float(scale[(f & 7) * 2 + (f >> 3)]);
}

// ---- the product ----------------------------------------------------------------
// One CTA of 16 warps per SM takes an equal share of the tiles.  Its x is staged
// in shared memory once, as columns of the tensor cores' B operand (features on m,
// rows of x on n), in a form that keeps every x' to its own 24 bits: a column whose
// codes are 0 at a row's large values must not inherit their step.
//   NP = 8, 4, 2  int8: x as a fixed-point number below a power of two over the
//           row's largest, one column for each of its bytes, NP bytes in an n tile.
//           Codes times bytes are summed exactly in int32, and unpacking eight codes
//           costs three instructions.  Up to four rows have eight bytes (61 bits, so
//           that an x' 2^37 below the largest still has its own 24); groups of three or
//           four fp16 rows with LayerNorm six (46 bits, more than fp16 spans).  Four bytes took 6.9 us for 4 rows
//           of 1600 x 6400 with LayerNorm, where eight take 7.9, and 14.7 and 18.1 for
//           1600 x 50257, but left 10 bits of a value 2^20 below the largest.  Leaving the
//           lower bytes out where no x' needs them, by a second loop or a second pass, cost
//           every call 0.6 us or more, or calls with one tiny value 3 us.
//   NP = 3  three bf16 parts: the upper 8 bits of 2^-16 x (which keeps sums of its
//           largest values finite), of the rest and of what that leaves, cut off, not
//           rounded, so that they add up to x.  A part has 8 rows in an n tile;
//           each part has its own sums over 32 or 64 rows of W, joined smallest first.
//           Eight codes cost eleven instructions.
//   NP = 1  fp16 x as it is, nine instructions for eight codes.
//
// The CTA's (tile, chunk) units are cut into 16 equal ranges, one per warp, so
// that each warp streams one contiguous piece of the packed matrix whatever the
// shape, through a ring of its own in shared memory (cp.async; registers as the
// ring left at most a few loads in flight).  The weights are read once, and
// nothing else is large.  A tile that crosses warps is summed in warp order, so
// the bits do not depend on timing.
constexpr int kQ4Warps = 16, kQ4Threads = 32 * kQ4Warps;
constexpr int kMaxTiles = 32;              // tiles of a CTA summed at a time
constexpr int kQ4Smem = 220 * 1024;

// One stage: a chunk of each of TP feature tiles.
template <int NT, int TP>
struct Q4Ring {
    static constexpr int kStages = TP == 1 ? 8 : NT > 1 ? 4 : 5;
};

struct Q4Args {
    const void *x;
    const unsigned char *packed;
    const float *bias, *gamma, *beta;
    const void *residual;
    void *y;
    int M, gelu;
    int copy;                              // fp16 rows of x can be copied 16 bytes at a time
    int rows;                              // rows of x of a CTA
    int slice;                             // chunks of x staged at a time
    int most;                              // tiles (of TP feature tiles) summed at a time
    int share, extra;                      // tiles of a CTA, CTAs that have one more
    // where LayerNorm's weights of a slice are staged (bytes; 0: nowhere)
    int ln;
};

// p[k .. k + 3] as fp32, 0 past K; VEC: in one load (K a multiple of 4, p aligned to it)
template <bool VEC, typename T>
__device__ __forceinline__ float4 load_4(const T *p, int k, int K) {
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (VEC) {
        if (k < K) {
            if (sizeof(T) == 2) {
                const uint2 u = *reinterpret_cast<const uint2 *>(p + k);
                const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&u.x));
                const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&u.y));
                v = make_float4(a.x, a.y, b.x, b.y);
            } else {
                v = *reinterpret_cast<const float4 *>(p + k);
            }
        }
    } else {
        if (k < K) v.x = tof(p[k]);
        if (k + 1 < K) v.y = tof(p[k + 1]);
        if (k + 2 < K) v.z = tof(p[k + 2]);
        if (k + 3 < K) v.w = tof(p[k + 3]);
    }
    return v;
}

__device__ __forceinline__ void mma16816_bf16(float (&c)[4], const unsigned (&w)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(b0), "r"(b1));
}
// The same onto zeros.
__device__ __forceinline__ void mma16816_bf16_first(float (&c)[4], const unsigned (&w)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

// Two codes as two fp16 of 1024 + (16 times, for upper nibbles) code + 8: flipping a
// two's complement nibble's sign bit adds 8, and 0x6400 | n is 1024 + n.
__device__ __forceinline__ __half2 nibbles(unsigned w, unsigned mask, unsigned flip) {
    unsigned r;
    asm("lop3.b32 %0, %1, %2, %3, 0x6A;" : "=r"(r) : "r"(w), "r"(mask), "r"(flip));   // (w & mask) ^ flip
    return *reinterpret_cast<__half2 *>(&r);
}
__device__ __forceinline__ unsigned bits(__half2 v) { return *reinterpret_cast<unsigned *>(&v); }
__device__ __forceinline__ void codes_to_half(unsigned w, unsigned (&f)[4]) {
    const __half2 low = __half2half2(__ushort_as_half((unsigned short)0x6408));   // 1032
    const __half2 sixteenth = __half2half2(__ushort_as_half((unsigned short)0x2c00)), up = __half2half2(__ushort_as_half((unsigned short)0xd480));   // -72
    f[0] = bits(__hfma2(nibbles(w, 0x00f000f0u, 0x64806480u), sixteenth, up));
    f[1] = bits(__hsub2(nibbles(w, 0x000f000fu, 0x64086408u), low));
    w >>= 8;
    f[2] = bits(__hfma2(nibbles(w, 0x00f000f0u, 0x64806480u), sixteenth, up));
    f[3] = bits(__hsub2(nibbles(w, 0x000f000fu, 0x64086408u), low));
}

// As bf16 pairs: 0x4300 | n is 128 + n.
__device__ __forceinline__ void codes_to_bf16(unsigned w, unsigned (&f)[4]) {
    const __nv_bfloat162 low = __bfloat162bfloat162(__ushort_as_bfloat16((unsigned short)0x4308));   // 136
    auto pair = [&](unsigned v) {
        unsigned r;
        asm("lop3.b32 %0, %1, %2, %3, 0x6A;" : "=r"(r) : "r"(v), "r"(0x000f000fu), "r"(0x43084308u));   // (v & mask) ^ flip
        const __nv_bfloat162 p = __hsub2(*reinterpret_cast<__nv_bfloat162 *>(&r), low);
        return *reinterpret_cast<const unsigned *>(&p);
    };
    f[0] = pair(w >> 4);
    f[1] = pair(w);
    f[2] = pair(w >> 12);
    f[3] = pair(w >> 8);
}

// Sum of v over the `n` warps of a row, a power of two that begins at warp `w0`: every lane gets it.
// `scratch` must not be in use by an earlier reduction.
__device__ __forceinline__ float row_sum(float v, float *scratch, int w0, int n) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (n > 1) {
        if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
        __syncthreads();
        v = scratch[w0 + (threadIdx.x & (n - 1))];
        for (int o = n >> 1; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    return v;
}
__device__ __forceinline__ unsigned row_largest(unsigned v, unsigned *scratch, int w0, int n) {
    v = __reduce_max_sync(0xffffffffu, v);
    if (n > 1) {
        if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
        __syncthreads();
        v = __reduce_max_sync(0xffffffffu, scratch[w0 + (threadIdx.x & (n - 1))]);
    }
    return v;
}

// Bytes of a staged column: 64 past a multiple of 128, so that eight columns' reads meet no bank twice.
template <int NP>
__host__ __device__ __forceinline__ int x_stride(int slice) {
    return NP == 8 || NP == 4 || NP == 2 ? (slice * kChunk + 127) / 128 * 128 + 64 : slice * kChunk * 2 + 64;
}
// Rows of x that the columns hold, and columns for them.
template <int NT, int NP>
constexpr int kRowsHeld = NP == 8 || NP == 4 || NP == 2 ? 8 / NP : 8 * NT;
template <int NT, int NP>
constexpr int kColumns = NP == 3 ? 24 * NT : 8 * NT;

// NT n tiles of 8 columns (of each of three parts where NP is 3), TP feature tiles that share an operand of x, the form
// NP of x (above), PC scale groups a chunk.
template <typename T, bool VEC, int NT, int TP, int NP, int PC>
__global__ void __launch_bounds__(kQ4Threads, 1) q4_matvec_kernel(Q4Args a, Q4Shape sh) {
    constexpr int S = Q4Ring<NT, TP>::kStages, CB = 512 + 32 * PC;
    constexpr bool INT = NP == 8 || NP == 4 || NP == 2, BF = NP == 3, STAGE_LN = VEC && BF;
    constexpr int kHeld = INT ? 4 : 8;                        // groups of four x that a thread reads once
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float sums[kQ4Warps], squares[kQ4Warps], up_s[G2_Q4_MAX_ROWS];
    __shared__ unsigned peaks[kQ4Warps];
    __shared__ float2 row_stats[G2_Q4_MAX_ROWS];
    __shared__ unsigned char range_s[kMaxTiles][2];
    constexpr int kPairs = INT ? NT * NP / 2 : 1;                 // pairs of bytes of an x
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    pdl_wait();
    pdl_launch();
    const int row0 = blockIdx.y * a.rows, M = min(a.rows, a.M - row0), K = sh.K;   // other rows are other CTAs'
    const T *x_rows = static_cast<const T *>(a.x) + (size_t)row0 * K;
    const T *residual = a.residual ? static_cast<const T *>(a.residual) + (size_t)row0 * sh.N : nullptr;
    T *y = static_cast<T *>(a.y) + (size_t)row0 * sh.N;
    const int stride = x_stride<NP>(a.slice);                     // bytes of a column
    unsigned char *ring = smem + (size_t)warp * S * TP * CB;      // [stage][TP] chunks
    unsigned char *xs = smem + (size_t)kQ4Warps * S * TP * CB;    // [columns][stride]
    float *pieces = reinterpret_cast<float *>(xs + (size_t)kColumns<NT, NP> * stride);   // [tiles + warps][M][16 TP]
    float *total = pieces + (size_t)(a.most + kQ4Warps) * M * 16 * TP;                // [M][tiles][16 TP], only with slices
    const unsigned ring_addr = smem_addr(ring);
    const int b = blockIdx.x;                                     // tiles of TP feature tiles: a.share, or one more
    const int tile0 = b * a.share + min(b, a.extra), tile1 = tile0 + a.share + (b < a.extra);
    // warps of a row of x in the passes over it
    int wpr = kQ4Warps;
    while (wpr * M > kQ4Warps && wpr > 1) wpr >>= 1;
    const int w0 = warp / wpr * wpr;
    const int first = ((warp - w0) * 32 + lane) * 4, step = wpr * 128;

    for (int tile = tile0; tile < tile1; tile += a.most) {
        const int R = min(a.most, tile1 - tile);
        for (int c0 = 0; c0 < sh.chunks; c0 += a.slice) {
            const int nc = min(a.slice, sh.chunks - c0);          // chunks of this slice
            const int U = R * nc;                                 // units, in 16 ranges, or one a warp
            auto range_begin = [&](int w) { return U < kQ4Warps ? min(w, U) : w * U / kQ4Warps; };
            const int u0 = range_begin(warp), u1 = range_begin(warp + 1), r_first = u0 / nc, c_first = u0 - r_first * nc;

            const bool stage_x = sh.chunks > a.slice || tile == tile0;
            if (NP == 1 && a.copy && stage_x) {                   // x as it is, ahead of the codes
                const int per_row = nc * (kChunk / 8);
                for (int i = tid; i < M * per_row; i += kQ4Threads) {
                    const int m = i / per_row, k = i % per_row * 8, left = K - c0 * kChunk - k;
                    cp_async16(smem_addr(xs + m * stride + 2 * k),
                               reinterpret_cast<const __half *>(x_rows) + (size_t)m * K + (left > 0 ? c0 * kChunk + k : 0), left > 0 ? 16 : 0);
                }
            }
            if (STAGE_LN && a.ln && stage_x) {
                for (int i = tid; i < nc * (kChunk / 2); i += kQ4Threads) {
                    const int second = i >= nc * (kChunk / 4), k = (i - second * nc * (kChunk / 4)) * 4, at = c0 * kChunk + k;
                    cp_async16(smem_addr(smem + a.ln) + 16 * i, (second ? a.beta : a.gamma) + (at < K ? at : 0), at < K ? 16 : 0);
                }
            }
            cp_commit();

            // ---- the first copies of the codes
            const size_t tile_bytes = (size_t)sh.chunks * CB;
            const unsigned char *src = a.packed + sh.at((tile + r_first) * TP, c0 + c_first) + lane * 16;
            int left = u1 - u0, lc = nc - c_first, put = 0;       // units to copy, chunks left of the tile, slot
            auto issue = [&]() {
                if (left > 0) {
                    const unsigned slot = ring_addr + put * (TP * CB) + lane * 16;
#pragma unroll
                    for (int x = 0; x < TP; ++x) {
                        cp_async16(slot + x * CB, src + x * tile_bytes, 16);
                        if (lane < 2 * PC) cp_async16(slot + x * CB + 512, src + x * tile_bytes + 512, 16);
                    }
                    src += CB;
                    if (--lc == 0) {
                        lc = nc;
                        src += TP * tile_bytes - nc * CB;
                    }
                    put = put + 1 == S ? 0 : put + 1;
                    --left;
                }
                cp_commit();
            };
#pragma unroll
            for (int p = 0; p < S - 1; ++p) issue();

            // ---- x of this slice, once
            if (stage_x && !(NP == 1 && a.copy)) {
                const int k0 = c0 * kChunk, kn = nc * kChunk;
                const int m = warp / wpr;                         // wpr M <= 16: every row has its warps; columns past M rows keep what they hold
                const bool live = m < M;
                const T *row = x_rows + (size_t)(live ? m : 0) * K;
                if constexpr (NP == 1) {
                    for (int k = live ? first : kn; k < kn; k += step) {
                        const float4 v = load_4<VEC>(row, k0 + k, K);
                        uint2 o;
                        o.x = bits(__floats2half2_rn(v.x, v.y));
                        o.y = bits(__floats2half2_rn(v.z, v.w));
                        *reinterpret_cast<uint2 *>(xs + m * stride + 2 * k) = o;
                    }
                } else {
                    // groups past the slice are skipped by whole warps; few rows have registers for LayerNorm's weights too
                    float4 held[kHeld], ga[INT ? kHeld : 1], be[INT ? kHeld : 1];
#pragma unroll
                    for (int i = 0; i < kHeld; ++i)
                        if (i * step < kn) {
                            const int k = min(k0 + first + i * step, K);
                            held[i] = load_4<VEC>(row, k, K);
                            if (INT && a.gamma) {
                                ga[INT ? i : 0] = load_4<VEC>(a.gamma, k, K);
                                be[INT ? i : 0] = load_4<VEC>(a.beta, k, K);
                            }
                        }
                    if (STAGE_LN && a.ln) {
                        cp_wait<S - 1>();
                        __syncthreads();
                    }
                    auto weight = [&](const float *p, int second, int k) -> float4 {   // p[k0 + k ...], 0 past the slice
                        if (!STAGE_LN || !a.ln) return load_4<VEC>(p, min(k0 + k, K), K);
                        return k < kn ? *reinterpret_cast<const float4 *>(smem + a.ln + 4 * (second * kn + k)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    };
                    float mu = 0.0f, rstd = 1.0f;
                    if (a.gamma) {
                        if (c0 == 0 && tile == tile0) {
                            const bool in_regs = kn >= K && K <= kHeld * step;
                            float s = 0.0f, q = 0.0f;
                            if (in_regs) {
#pragma unroll
                                for (int i = 0; i < kHeld; ++i)
                                    if (i * step < kn) s += (held[i].x + held[i].y) + (held[i].z + held[i].w);
                            } else {
#pragma unroll 4
                                for (int k = first; k < K; k += step) {
                                    const float4 v = load_4<VEC>(row, k, K);
                                    s += (v.x + v.y) + (v.z + v.w);
                                }
                            }
                            mu = row_sum(s, sums, w0, wpr) / K;
                            auto square = [&](const float4 &v, int k) {
                                const float d0 = v.x - mu, d1 = v.y - mu, d2 = v.z - mu, d3 = v.w - mu;
                                if (VEC) {
                                    if (k < K) q += fmaf(d0, d0, d1 * d1) + fmaf(d2, d2, d3 * d3);
                                } else {
                                    if (k < K) q = fmaf(d0, d0, q);
                                    if (k + 1 < K) q = fmaf(d1, d1, q);
                                    if (k + 2 < K) q = fmaf(d2, d2, q);
                                    if (k + 3 < K) q = fmaf(d3, d3, q);
                                }
                            };
                            if (in_regs) {
#pragma unroll
                                for (int i = 0; i < kHeld; ++i)
                                    if (i * step < kn) square(held[i], first + i * step);
                            } else {
#pragma unroll 4
                                for (int k = first; k < K; k += step) square(load_4<VEC>(row, k, K), k);
                            }
                            rstd = rsqrtf(row_sum(q, squares, w0, wpr) / K + 1e-5f);
                            if (live && first == 0) row_stats[m] = make_float2(mu, rstd);
                        } else {
                            mu = row_stats[live ? m : 0].x;
                            rstd = row_stats[live ? m : 0].y;
                        }
                    }
                    auto norm = [&](const float4 &v, const float4 &gv, const float4 &bv) -> float4 {
                        return make_float4(fmaf((v.x - mu) * rstd, gv.x, bv.x), fmaf((v.y - mu) * rstd, gv.y, bv.y),
                                           fmaf((v.z - mu) * rstd, gv.z, bv.z), fmaf((v.w - mu) * rstd, gv.w, bv.w));
                    };
                    auto value = [&](int k) -> float4 {           // x'[m][k .. k + 3], 0 past K
                        const float4 v = load_4<VEC>(row, k0 + k, K);
                        return a.gamma ? norm(v, weight(a.gamma, 0, k), weight(a.beta, 1, k)) : v;
                    };
                    auto normed = [&](int i) -> float4 {          // held[i] after LayerNorm; past K: 0 * 0 + 0
                        if (!a.gamma) return held[i];
                        const int k = first + i * step;
                        return INT ? norm(held[i], ga[INT ? i : 0], be[INT ? i : 0]) : norm(held[i], weight(a.gamma, 0, k), weight(a.beta, 1, k));
                    };
                    if constexpr (BF) {
                        auto put = [&](const float4 &v, int k) {
                            float r[4] = {v.x * 0x1p-16f, v.y * 0x1p-16f, v.z * 0x1p-16f, v.w * 0x1p-16f};
                            unsigned char *o = xs + m * stride + 2 * k;
#pragma unroll
                            for (int p = 0; p < 3; ++p, o += 8 * NT * stride) {
                                const uint2 w = make_uint2(__byte_perm(__float_as_uint(r[0]), __float_as_uint(r[1]), 0x7632),
                                                           __byte_perm(__float_as_uint(r[2]), __float_as_uint(r[3]), 0x7632));
                                *reinterpret_cast<uint2 *>(o) = w;
#pragma unroll
                                for (int j = 0; j < 4; ++j) r[j] -= __uint_as_float(__float_as_uint(r[j]) & 0xffff0000u);
                            }
                        };
#pragma unroll
                        for (int i = 0; i < kHeld; ++i)
                            if (i * step < kn) {
                                const float4 v = normed(i);
                                if (live && first + i * step < kn) put(v, first + i * step);
                            }
#pragma unroll 4
                        for (int k = live ? first + kHeld * step : kn; k < kn; k += step) put(value(k), k);
                    } else {
                        // as integers: NaN above infinity above finite
                        unsigned peak = 0;
                        auto measure = [&](const float4 &v) {
                            const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                            for (int j = 0; j < 4; ++j) peak = max(peak, __float_as_uint(x[j]) & 0x7fffffffu);
                        };
#pragma unroll
                        for (int i = 0; i < kHeld; ++i)
                            if (i * step < kn) {
                                held[i] = normed(i);
                                measure(held[i]);
                            }
#pragma unroll 4
                        for (int k = first + kHeld * step; k < kn; k += step) measure(value(k));
                        peak = row_largest(peak, peaks, w0, wpr);
                        // 2^e <= the largest < 2^(e + 1): 29 bits below it are the upper four bytes' unit, and the codes are 16 times theirs
                        const int e = max(-96, min(127, (int)(peak >> 23) - 127));
                        const float down = __uint_as_float((unsigned)(127 + 29 - e) << 23);
                        if (live && first == 0)
                            up_s[m] = peak >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __uint_as_float((unsigned)(127 + e) << 23) * 0x1p-33f;
                        auto put = [&](const float4 &v, int k) {
                            // rows k, k + 2, k + 1, k + 3 of a column, the most significant bytes first
                            unsigned char *o = xs + m * NP * stride + (k & ~63) + ((k >> 3) & 3) * 16 + ((k >> 5) & 1) * 8 + (k & 7);
                            auto column = [&](int b) { return reinterpret_cast<unsigned *>(o + (b / NP * 8 + b % NP) * stride); };
                            float x[4] = {v.x * down, v.y * down, v.z * down, v.w * down};
#pragma unroll
                            for (int half = 0; half < (kPairs + 1) / 2; ++half) {
                                const bool two = kPairs == 3 && half == 1;   // two bytes, not four
                                unsigned q[4];
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    const int n = __float2int_rn(x[j]);
                                    x[j] = (x[j] - (float)n) * (kPairs == 3 ? 0x1p15f : 0x1p31f);   // both exact: n has at most the bits of x
                                    // signed bytes: adding 128 to each of the lower ones carries into the next
                                    q[j] = two ? ((unsigned)n + 0x0080u) ^ 0x0080u : ((unsigned)n + 0x00808080u) ^ 0x00808080u;
                                }
                                const unsigned l01 = __byte_perm(q[0], q[2], 0x5140), l23 = __byte_perm(q[1], q[3], 0x5140);   // bytes 0 and 1 of both
                                const unsigned h01 = __byte_perm(q[0], q[2], 0x7362), h23 = __byte_perm(q[1], q[3], 0x7362);   // bytes 2 and 3
                                if (!two) {
                                    *column(4 * half) = __byte_perm(h01, h23, 0x7632);
                                    *column(4 * half + 1) = __byte_perm(h01, h23, 0x5410);
                                }
                                *column(4 * half + (two ? 0 : 2)) = __byte_perm(l01, l23, 0x7632);
                                *column(4 * half + (two ? 1 : 3)) = __byte_perm(l01, l23, 0x5410);
                            }
                        };
#pragma unroll
                        for (int i = 0; i < kHeld; ++i)
                            if (i * step < kn && live && first + i * step < kn) put(held[i], first + i * step);
#pragma unroll 4
                        for (int k = live ? first + kHeld * step : kn; k < kn; k += step) put(value(k), k);
                    }
                }
            }
            if (tid < R) {                                        // the warps that have units of each tile
                const int W = min(kQ4Warps, U);                   // unit u is warp ((u + 1) W - 1) / U's
                range_s[tid][0] = (unsigned char)(((tid * nc + 1) * W - 1) / U);
                range_s[tid][1] = (unsigned char)(((tid + 1) * nc * W - 1) / U);
            }
            cp_wait<S - 1>();                                     // x, where it was copied
            __syncthreads();

            // ---- the warp's units
            constexpr int kTot = INT ? 2 : 4;
            float tot[TP][NT][kTot];
#pragma unroll
            for (int x = 0; x < TP; ++x)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < kTot; ++i) tot[x][n][i] = 0.0f;
            int r = r_first, c = nc - c_first;                    // tile, chunks left of it
            constexpr int kStep = INT ? kChunk : 2 * kChunk;      // bytes of a column in a chunk
            const unsigned char *xk = xs + g * stride + t * 16 + c_first * kStep;
            const unsigned char *slot = ring;
            for (int u = u0; u < u1; ++u) {
                cp_wait<S - 2>();
                __syncwarp();
                issue();
                if constexpr (BF) {
                    constexpr bool BOTH = PC == 1;                // sums over 64 rows, or over a group of 32
                    uint4 w[TP];
#pragma unroll
                    for (int x = 0; x < TP; ++x) w[x] = *reinterpret_cast<const uint4 *>(slot + x * CB + lane * 16);
                    float acc[TP][3][NT][4];
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint4 xv[3][NT];
#pragma unroll
                        for (int p = 0; p < 3; ++p)
#pragma unroll
                            for (int n = 0; n < NT; ++n)
                                xv[p][n] = *reinterpret_cast<const uint4 *>(xk + (p * NT + n) * 8 * stride + half * 64);
#pragma unroll
                        for (int x = 0; x < TP; ++x) {
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                unsigned f[4];
                                codes_to_bf16(half ? (i ? w[x].w : w[x].z) : (i ? w[x].y : w[x].x), f);
#pragma unroll
                                for (int p = 0; p < 3; ++p)
#pragma unroll
                                    for (int n = 0; n < NT; ++n) {
                                        const unsigned b0 = i ? xv[p][n].z : xv[p][n].x, b1 = i ? xv[p][n].w : xv[p][n].y;
                                        if (i == 0 && (half == 0 || !BOTH)) mma16816_bf16_first(acc[x][p][n], f, b0, b1);
                                        else mma16816_bf16(acc[x][p][n], f, b0, b1);
                                    }
                            }
                            if (half == 1 || !BOTH) {             // the group's sum, scaled
                                const unsigned s = *reinterpret_cast<const unsigned *>(slot + x * CB + 512 + (PC == 2 ? half * 32 : 0) + g * 4);
                                const float lo = __uint_as_float(s << 16), hi = __uint_as_float(s & 0xffff0000u);
#pragma unroll
                                for (int n = 0; n < NT; ++n)
#pragma unroll
                                    for (int j = 0; j < 4; ++j)
                                        tot[x][n][j] = fmaf((acc[x][2][n][j] + acc[x][1][n][j]) + acc[x][0][n][j], j < 2 ? lo : hi, tot[x][n][j]);
                            }
                        }
                    }
                } else if constexpr (INT) {
                    uint4 xv[NT];
#pragma unroll
                    for (int n = 0; n < NT; ++n) xv[n] = *reinterpret_cast<const uint4 *>(xk + n * 8 * stride);
#pragma unroll
                    for (int x = 0; x < TP; ++x) {
                        const uint4 w = *reinterpret_cast<const uint4 *>(slot + x * CB + lane * 16);
                        const unsigned words[4] = {w.x, w.y, w.z, w.w};
                        unsigned sc[PC];
#pragma unroll
                        for (int i = 0; i < PC; ++i) sc[i] = *reinterpret_cast<const unsigned *>(slot + x * CB + 512 + i * 32 + g * 4);
                        int acc[NT][4];
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            if (i == 0 || PC == 2)
#pragma unroll
                                for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0;
                            const unsigned u0 = words[2 * i], u1 = words[2 * i + 1];
                            const unsigned f[4] = {u0 & 0xf0f0f0f0u, (u0 << 4) & 0xf0f0f0f0u, u1 & 0xf0f0f0f0u, (u1 << 4) & 0xf0f0f0f0u};
#pragma unroll
                            for (int n = 0; n < NT; ++n) mma16832(acc[n], f, i ? xv[n].z : xv[n].x, i ? xv[n].w : xv[n].y);
                            if (i == 1 || PC == 2) {          // the group's sums of two neighbouring bytes, below 2^29
                                const unsigned s = sc[PC == 2 ? i : 0];
                                const float lo = __uint_as_float(s << 16), hi = __uint_as_float(s & 0xffff0000u);
#pragma unroll
                                for (int n = 0; n < NT; ++n) {
                                    tot[x][n][0] = fmaf((float)(acc[n][0] * 256 + acc[n][1]), lo, tot[x][n][0]);
                                    tot[x][n][1] = fmaf((float)(acc[n][2] * 256 + acc[n][3]), hi, tot[x][n][1]);
                                }
                            }
                        }
                    }
                } else {
                    uint4 xv[NT][2];
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int half = 0; half < 2; ++half)
                            xv[n][half] = *reinterpret_cast<const uint4 *>(xk + n * 8 * stride + half * 64);
#pragma unroll
                    for (int x = 0; x < TP; ++x) {
                        const uint4 w = *reinterpret_cast<const uint4 *>(slot + x * CB + lane * 16);
                        const unsigned words[4] = {w.x, w.y, w.z, w.w};
                        unsigned sc[PC];
#pragma unroll
                        for (int i = 0; i < PC; ++i) sc[i] = *reinterpret_cast<const unsigned *>(slot + x * CB + 512 + i * 32 + g * 4);
                        float acc[NT][4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if (i == 0 || (PC == 2 && i == 2))
#pragma unroll
                                for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.0f;
                            unsigned f[4];
                            codes_to_half(words[i], f);
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                const uint4 &v = xv[n][i >> 1];
                                mma16816(acc[n], f, (i & 1) ? v.z : v.x, (i & 1) ? v.w : v.y);
                            }
                            if (i == 3 || (PC == 2 && i == 1)) {  // the group's sum, scaled
                                const unsigned s = sc[PC == 2 ? i >> 1 : 0];
                                const float lo = __uint_as_float(s << 16), hi = __uint_as_float(s & 0xffff0000u);
#pragma unroll
                                for (int n = 0; n < NT; ++n) {
                                    tot[x][n][0] = fmaf(acc[n][0], lo, tot[x][n][0]);
                                    tot[x][n][1] = fmaf(acc[n][1], lo, tot[x][n][1]);
                                    tot[x][n][2] = fmaf(acc[n][2], hi, tot[x][n][2]);
                                    tot[x][n][3] = fmaf(acc[n][3], hi, tot[x][n][3]);
                                }
                            }
                        }
                    }
                }
                slot = slot + TP * CB == ring + S * TP * CB ? ring : slot + TP * CB;
                xk += kStep;
                if (--c == 0 || u == u1 - 1) {                    // (this warp's part of) a tile is done
                    float *o = pieces + (size_t)(r + warp) * M * 16 * TP + g;
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int x = 0; x < TP; ++x) {
                            float (&v)[kTot] = tot[x][n];
                            if constexpr (INT) {                  // thread t has two bytes of each tile, the upper ones first
                                if (n > 0) break;
                                constexpr int kThreads = NP / 2;  // threads of a row
#pragma unroll
                                for (int i = 0; i < 2; ++i) {
                                    auto pair = [&](int j) -> float {   // of the row that begins with this thread
                                        if (j >= kPairs) return 0.0f;
                                        const float w = tot[x][j / kThreads][i];
                                        return j % kThreads ? __shfl_down_sync(0xffffffffu, w, j % kThreads) : w;
                                    };
                                    float all = pair(1);
                                    if (kPairs > 2) all = fmaf(pair(2), 0x1p-15f, all);
                                    if (kPairs > 3) all = fmaf(pair(3), 0x1p-31f, all);
                                    all = fmaf(pair(0), 65536.0f, all);
                                    const int m = t / kThreads;
                                    if (m < M && t % kThreads == 0) o[m * 16 * TP + x * 16 + 8 * i] = all;
                                }
                            } else {
#pragma unroll
                                for (int i = 0; i < kTot; ++i) {
                                    const int m = n * 8 + 2 * t + (i & 1);
                                    if (m < M) o[m * 16 * TP + x * 16 + (i >> 1) * 8] = v[i];
                                }
                            }
                        }
#pragma unroll
                    for (int x = 0; x < TP; ++x)
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int i = 0; i < kTot; ++i) tot[x][n][i] = 0.0f;
                    c = nc;
                    xk -= nc * kStep;
                    ++r;
                }
            }
            cp_wait<0>();
            __syncthreads();

            // ---- sums over the warps of each tile, in order; after the last slice bias, GELU, residual
            // (four rows, a tile) at a time: 32 features of one item, or 16 of two, a warp
            constexpr int kPer = 2 / TP, kRows = INT ? 1 : 4;
            const int f = lane % (16 * TP), row_groups = (M + kRows - 1) / kRows;
            int mg = 0, rr = warp * kPer + lane / (16 * TP);
            for (;; rr += kQ4Warps * kPer) {
                for (; rr >= R && mg < row_groups; rr -= R) ++mg;
                if (mg >= row_groups) break;
                const int n = (tile + rr) * 16 * TP + f, m0 = mg * kRows, wa = range_s[rr][0], wb = range_s[rr][1];
                const bool last = c0 + nc == sh.chunks, there = last && n < sh.N;
                const float bias = there && a.bias ? a.bias[n] : 0.0f;
                float v[kRows], res[kRows];
#pragma unroll
                for (int j = 0; j < kRows; ++j) {
                    v[j] = 0.0f;
                    res[j] = there && residual && m0 + j < M ? tof(residual[(size_t)(m0 + j) * sh.N + n]) : 0.0f;
                }
                const float *o = pieces + ((rr + wa) * M + m0) * 16 * TP + f;
                for (int x = wa; x <= wb; ++x, o += M * 16 * TP)
#pragma unroll
                    for (int j = 0; j < kRows; ++j)
                        if (kRows == 1 || m0 + j < M) v[j] += o[j * 16 * TP];
#pragma unroll
                for (int j = 0; j < kRows; ++j) {
                    const int m = m0 + j;
                    if (m >= M) break;
                    float *so_far = total + (m * R + rr) * 16 * TP + f;
                    if (INT) v[j] *= up_s[m];
                    if (BF) v[j] *= 65536.0f;
                    if (c0 > 0) v[j] += *so_far;
                    if (!last) *so_far = v[j];
                    if (there) {
                        v[j] += bias;
                        if (a.gelu) v[j] = gelu_f(v[j]);
                        if (residual) v[j] += res[j];
                        y[(size_t)m * sh.N + n] = fromf<T>(v[j]);
                    }
                }
            }
            __syncthreads();
        }
    }
}

template <typename T, bool VEC, int NT, int TP, int NP, int PC>
int launch_q4(Q4Args a, const Q4Shape &sh, cudaStream_t st) {
    auto kernel = q4_matvec_kernel<T, VEC, NT, TP, NP, PC>;
    const int ntiles = sh.tiles / TP, grid = std::min(sm_count(), ntiles);
    a.share = ntiles / grid;
    a.extra = ntiles % grid;
    a.most = std::min((ntiles + grid - 1) / grid, kMaxTiles / TP);
    // x in equal slices that fit beside the ring and the sums
    const size_t ring = (size_t)kQ4Warps * Q4Ring<NT, TP>::kStages * TP * sh.chunk_bytes, tile = (size_t)std::min(a.M, a.rows) * 16 * TP * 4;
    size_t sums = (a.most + kQ4Warps) * tile;
    auto bytes = [&](int slice) { return ring + (size_t)kColumns<NT, NP> * x_stride<NP>(slice) + sums; };
    a.slice = sh.chunks;
    if (bytes(a.slice) > kQ4Smem) {
        sums += a.most * tile;
        int slices = 2;
        while (bytes((sh.chunks + slices - 1) / slices) > kQ4Smem) ++slices;   // ends: one chunk fits
        a.slice = (sh.chunks + slices - 1) / slices;
    }
    size_t smem = bytes(a.slice);
    // More rows have no registers for LayerNorm's weights: beside x, where there is room (8 rows of 1600 x 6400: 10.1 us without)
    a.ln = 0;
    if (VEC && NP == 3 && a.gamma && smem + a.slice * kChunk * 8 <= kQ4Smem) {
        a.ln = (int)smem;
        smem += a.slice * kChunk * 8;
    }
    // the most that any call uses, so that calls from several host threads do not undo each other's
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kQ4Smem) != cudaSuccess)
        return arg_error(G2_ERR_CUDA, "g2k_matvec_q4", cudaGetErrorString(cudaGetLastError()));
    return launch_status("g2k_matvec_q4", launch_pdl(kernel, dim3(grid, (a.M + a.rows - 1) / a.rows), dim3(kQ4Threads), smem, st, a, sh));
}

// `rows` rows of x to a CTA
template <typename T, bool VEC, int NT, int TP, int NP>
int launch_q4(Q4Args a, const Q4Shape &sh, int rows, cudaStream_t st) {
    a.rows = std::min(rows, kRowsHeld<NT, NP>);
    return sh.per_chunk == 2 ? launch_q4<T, VEC, NT, TP, NP, 2>(a, sh, st) : launch_q4<T, VEC, NT, TP, NP, 1>(a, sh, st);
}

template <typename T, bool VEC>
int launch_q4(const Q4Args &a, const Q4Shape &sh, cudaStream_t st) {
    // Two feature tiles share each operand of x, which halves its reads and the loop's own instructions;
    // matrices of fewer pairs than SMs are better spread one by one.
    const int sms = sm_count();
    const bool one = sh.tiles / 2 < sms;
    // Rows in groups of 2, 4 or 8: the fewest that one CTA per SM still holds, since staging x is most of a
    // narrow matrix's time (16 rows of 3974 x 83: 27 us in groups of 8, 5.8 in groups of 2), else as few groups as can be.
    const auto fits = [&](int rows) { return sh.tiles * ((a.M + rows - 1) / rows) <= sms; };
    if constexpr (sizeof(T) == 2)
        if (!a.gamma && a.M > 2 && !(a.M > 8 && fits(2)))
            return a.M > 8 ? launch_q4<T, VEC, 2, 2, 1>(a, sh, 16, st)
                 : one     ? launch_q4<T, VEC, 1, 1, 1>(a, sh, 8, st) : launch_q4<T, VEC, 1, 2, 1>(a, sh, 8, st);
    constexpr int kFour = sizeof(T) == 4 ? 4 : 3;   // n tiles of four rows' bytes
    if (a.M == 1) return one ? launch_q4<T, VEC, 1, 1, 8>(a, sh, 1, st) : launch_q4<T, VEC, 1, 2, 8>(a, sh, 1, st);
    if (a.M == 2 || fits(2)) return one ? launch_q4<T, VEC, 2, 1, 4>(a, sh, 2, st) : launch_q4<T, VEC, 2, 2, 4>(a, sh, 2, st);
    if (a.M <= 4 || fits(4)) return one ? launch_q4<T, VEC, kFour, 1, 2>(a, sh, 4, st) : launch_q4<T, VEC, kFour, 2, 2>(a, sh, 4, st);
    // Groups of eight: sixteen rows at once would leave room for half as much of x.  Two groups side by side
    // fill the SMs with pairs of tiles as well (16 rows of 1600 x 1600: 6.4 us, tile by tile 10.8).
    return one && a.M <= 8 ? launch_q4<T, VEC, 1, 1, 3>(a, sh, 8, st) : launch_q4<T, VEC, 1, 2, 3>(a, sh, 8, st);
}

bool bad_shape(int N, int K, int group) {
    return N < 1 || K < 1 || K > G2_Q4_MAX_K || (group != 32 && group != 64 && group != 128) ||
           (long long)N + 2 * kTile > 0x7fffffff;
}

}  // namespace

}  // namespace g2

using namespace g2;

extern "C" size_t g2k_q4_bytes(int N, int K, int group) {
    return bad_shape(N, K, group) ? 0 : Q4Shape(N, K, group).bytes();
}

static int check_packed(const char *who, const void *packed, int N, int K, int group) {
    if (group != 32 && group != 64 && group != 128) return arg_error(G2_ERR_ARG, who, "group must be 32, 64 or 128");
    if (bad_shape(N, K, group)) return arg_error(G2_ERR_RANGE, who, "need N >= 1 and 1 <= K <= 32768");
    if (!aligned(packed, 256)) return arg_error(G2_ERR_ARG, who, "packed is not 256-byte aligned");
    return G2_OK;
}

extern "C" int g2k_q4_pack(const void *W, int dtype, int transposed, void *packed, int N, int K, int group, void *stream) {
    const char *who = "g2k_q4_pack";
    if (!W || !packed) return arg_error(G2_ERR_ARG, who, "null argument");
    if (dtype != G2_F32 && dtype != G2_F16) return arg_error(G2_ERR_ARG, who, "bad dtype");
    int rc;
    if ((rc = check_packed(who, packed, N, K, group))) return rc;
    if (!aligned(W, dtype == G2_F32 ? 4 : 2)) return arg_error(G2_ERR_ARG, who, "W is not aligned to its elements");
    if ((rc = check_device_ptrs(who, {W, packed}))) return rc;
    const Q4Shape sh(N, K, group);
    unsigned char *out = static_cast<unsigned char *>(packed);
    const dim3 grid(sh.tiles, (sh.chunks * kChunk + group - 1) / group);   // groups past K too: their codes are 0
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == G2_F32)
        q4_pack_kernel<float><<<grid, kPackThreads, 0, st>>>(static_cast<const float *>(W), transposed, out, sh);
    else
        q4_pack_kernel<__half><<<grid, kPackThreads, 0, st>>>(static_cast<const __half *>(W), transposed, out, sh);
    return launch_status(who);
}

extern "C" int g2k_q4_unpack(const void *packed, float *W, int N, int K, int group, void *stream) {
    const char *who = "g2k_q4_unpack";
    if (!W || !packed) return arg_error(G2_ERR_ARG, who, "null argument");
    int rc;
    if ((rc = check_packed(who, packed, N, K, group))) return rc;
    if ((rc = check_device_ptrs(who, {W, packed}))) return rc;
    const Q4Shape sh(N, K, group);
    const long long blocks = ((long long)K * N + 255) / 256;
    if (blocks > 0x7fffffffLL) return arg_error(G2_ERR_RANGE, who, "matrix too large");
    q4_unpack_kernel<<<(unsigned)blocks, 256, 0, (cudaStream_t)stream>>>(static_cast<const unsigned char *>(packed), W, sh);
    return launch_status(who);
}

extern "C" int g2k_matvec_q4(const void *x, const void *packed, const float *bias, const void *residual, void *y, int dtype,
                             int M, int N, int K, int group, int apply_gelu, const float *ln_gamma, const float *ln_beta,
                             void *stream) {
    const char *who = "g2k_matvec_q4";
    if (!x || !packed || !y) return arg_error(G2_ERR_ARG, who, "null argument");
    if (dtype != G2_F32 && dtype != G2_F16) return arg_error(G2_ERR_ARG, who, "bad dtype");
    if ((ln_gamma == nullptr) != (ln_beta == nullptr)) return arg_error(G2_ERR_ARG, who, "ln_gamma and ln_beta go together");
    if (M < 1 || M > G2_Q4_MAX_ROWS) return arg_error(G2_ERR_RANGE, who, "need 1 <= M <= 16");
    int rc;
    if ((rc = check_packed(who, packed, N, K, group))) return rc;
    const size_t es = dtype == G2_F32 ? 4 : 2;
    if (!aligned(x, es) || !aligned(y, es) || !aligned(residual, es) || !aligned(bias, 4) || !aligned(ln_gamma, 4) ||
        !aligned(ln_beta, 4))
        return arg_error(G2_ERR_ARG, who, "an array is not aligned to its elements");
    if ((rc = check_device_ptrs(who, {x, packed, bias, residual, y, ln_gamma, ln_beta}))) return rc;
    const Q4Shape sh(N, K, group);
    const bool vec = K % 4 == 0 && aligned(x, 4 * es) && aligned(ln_gamma, 16) && aligned(ln_beta, 16);
    const Q4Args a{x, static_cast<const unsigned char *>(packed), bias, ln_gamma, ln_beta, residual, y, M, apply_gelu,
                   dtype == G2_F16 && K % 8 == 0 && !ln_gamma && aligned(x, 16), 0, 0, 0, 0, 0};
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == G2_F32) return vec ? launch_q4<float, true>(a, sh, st) : launch_q4<float, false>(a, sh, st);
    return vec ? launch_q4<__half, true>(a, sh, st) : launch_q4<__half, false>(a, sh, st);
}
