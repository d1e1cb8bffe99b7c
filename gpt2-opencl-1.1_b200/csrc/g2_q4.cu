// g2_q4.cu -- weights in 4 bits: packing (g2k_q4_pack), reading back
// (g2k_q4_unpack) and the matrix-vector product on them (g2k_matvec_q4).
//
// W [K][N] is cut into groups of `group` rows of a column.  A group's scale is
// s = bf16(max|w| / 7) and its codes c = w / s rounded, in -7..7, so that
//   y[m][n] = sum_groups s[g][n] * sum_{k in g} x'[m][k] c[k][n].
//
// Packed layout, for tiles of 16 columns (features) and chunks of 64 rows:
//   codes  [tile][chunk][lane 0..31][4 words]   512 bytes a chunk
//   scales [tile][group][8][2] bf16             features g and g + 8 of a tile together
// Word s of lane (g = lane / 4, t = lane % 4) holds features g and g + 8 at rows
// 64 chunk + 16 s + 4 t + {0, 1, 2, 3}, as code + 8 in nibbles
//   0, 4: feature g,     rows +0, +1      1, 5: feature g + 8, rows +0, +1
//   2, 6: feature g,     rows +2, +3      3, 7: feature g + 8, rows +2, +3
// so that nibbles j and j + 4 are register j of the A operand of a 16 x 8 x 16
// tensor-core product whose k index is a permutation of the rows.  Rows past K
// and columns past N hold code 0.
#include <cuda_bf16.h>

#include "g2_args.h"
#include "g2_device.cuh"

namespace g2 {

namespace {

constexpr int kTile = 16, kChunk = 64;

struct Q4Shape {
    int N, K, group;
    int tiles, chunks, groups;   // groups cover the chunks (zero scales past K)
    long long scale_off;         // bytes from the codes to the scales
    __host__ __device__ Q4Shape(int N_, int K_, int group_) : N(N_), K(K_), group(group_) {
        tiles = (N + kTile - 1) / kTile;
        chunks = (K + kChunk - 1) / kChunk;
        groups = (chunks * kChunk + group - 1) / group;
        scale_off = ((long long)tiles * chunks * 512 + 255) / 256 * 256;
    }
    size_t bytes() const { return (size_t)scale_off + (size_t)tiles * groups * kTile * 2; }
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
__global__ void __launch_bounds__(kPackThreads) q4_pack_kernel(const T *W, int transposed, unsigned *codes,
                                                               __nv_bfloat16 *scales, Q4Shape sh) {
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
        const size_t o = ((size_t)tile * sh.groups + grp) * kTile + (t & 7) * 2 + (t >> 3);
        scales[o] = peak[t] >= 0x7f800000u ? __ushort_as_bfloat16(0x7fc0) : s;
    }
    __syncthreads();
    for (int i = t; i < sh.group * kTile; i += kPackThreads) {
        int f, k;
        at(i, f, k);
        const float s = step[f];
        int c = 0;
        if (s > 0.0f && peak[f] < 0x7f800000u) c = max(-7, min(7, round_quotient(load(f, k), s)));
        code[k][f] = (unsigned char)(c + 8);
    }
    __syncthreads();
    // 32 lanes per 16 rows
    for (int i = t; i < sh.group * 2; i += kPackThreads) {
        const int lane = i & 31, step16 = i >> 5, kk = k0 + step16 * 16;
        const int chunk = kk / kChunk, s = (kk % kChunk) / 16;
        if (chunk >= sh.chunks) continue;
        const int g = lane >> 2, r = step16 * 16 + (lane & 3) * 4;
        unsigned w = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int f = g + (j & 1) * 8, k = r + (j >> 1) * 2;
            w |= (unsigned)code[k][f] << (4 * j);
            w |= (unsigned)code[k + 1][f] << (4 * j + 16);
        }
        codes[(((size_t)tile * sh.chunks + chunk) * 32 + lane) * 4 + s] = w;
    }
}

__device__ __forceinline__ int q4_code(const unsigned *codes, const Q4Shape &sh, int k, int n) {
    const int f = n % kTile, kc = k % kChunk, r = kc & 3;
    const int lane = (f & 7) * 4 + ((kc >> 2) & 3);
    const unsigned w = codes[(((size_t)(n / kTile) * sh.chunks + k / kChunk) * 32 + lane) * 4 + kc / 16];
    const int nib = (f >> 3) + (r >> 1) * 2 + (r & 1) * 4;
    return (int)((w >> (4 * nib)) & 15u) - 8;
}

__device__ __forceinline__ float q4_scale(const __nv_bfloat16 *scales, const Q4Shape &sh, int k, int n) {
    const int f = n % kTile;
    return __bfloat162float(scales[((size_t)(n / kTile) * sh.groups + k / sh.group) * kTile + (f & 7) * 2 + (f >> 3)]);
}

__global__ void __launch_bounds__(256) q4_unpack_kernel(const unsigned *codes, const __nv_bfloat16 *scales, float *W,
                                                        Q4Shape sh) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long long)sh.K * sh.N) return;
    const int k = (int)(i / sh.N), n = (int)(i % sh.N);
    W[i] = q4_code(codes, sh, k, n) * q4_scale(scales, sh, k, n);
}

// The product, one warp per feature: each lane takes every 32nd row.
struct Q4Args {
    const void *x;
    const unsigned *codes;
    const __nv_bfloat16 *scales;
    const float *bias, *gamma, *beta;
    const void *residual;
    void *y;
    int M, gelu;
};

template <typename T>
__global__ void __launch_bounds__(256) q4_matvec_kernel(Q4Args a, Q4Shape sh) {
    __shared__ float mean_s[G2_Q4_MAX_ROWS], rstd_s[G2_Q4_MAX_ROWS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, K = sh.K;
    const T *x = static_cast<const T *>(a.x);
    if (a.gamma) {
        for (int m = warp; m < a.M; m += 8) {
            float s = 0.0f;
            for (int k = lane; k < K; k += 32) s += tof(x[(size_t)m * K + k]);
            for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            const float mu = s / K;
            float v = 0.0f;
            for (int k = lane; k < K; k += 32) {
                const float d = tof(x[(size_t)m * K + k]) - mu;
                v += d * d;
            }
            for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
            if (lane == 0) {
                mean_s[m] = mu;
                rstd_s[m] = rsqrtf(v / K + 1e-5f);
            }
        }
        __syncthreads();
    }
    const int n = blockIdx.x * 8 + warp;
    if (n >= sh.N) return;
    float acc[G2_Q4_MAX_ROWS] = {};
    for (int k = lane; k < K; k += 32) {
        const float w = q4_code(a.codes, sh, k, n) * q4_scale(a.scales, sh, k, n);
        const float ga = a.gamma ? a.gamma[k] : 0.0f, be = a.gamma ? a.beta[k] : 0.0f;
#pragma unroll
        for (int m = 0; m < G2_Q4_MAX_ROWS; ++m) {
            if (m >= a.M) break;
            float v = tof(x[(size_t)m * K + k]);
            if (a.gamma) v = (v - mean_s[m]) * rstd_s[m] * ga + be;
            acc[m] += v * w;
        }
    }
#pragma unroll
    for (int m = 0; m < G2_Q4_MAX_ROWS; ++m) {
        if (m >= a.M) break;
        float v = acc[m];
        for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane == 0) {
            if (a.bias) v += a.bias[n];
            if (a.gelu) v = gelu_f(v);
            const size_t i = (size_t)m * sh.N + n;
            if (a.residual) v += tof(static_cast<const T *>(a.residual)[i]);
            static_cast<T *>(a.y)[i] = fromf<T>(v);
        }
    }
}

bool bad_shape(int N, int K, int group) {
    return N < 1 || K < 1 || K > G2_Q4_MAX_K || (group != 32 && group != 64 && group != 128) ||
           ((long long)N + kTile - 1) / kTile > 0x7fffffff / kTile;
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
    unsigned *codes = static_cast<unsigned *>(packed);
    auto *scales = reinterpret_cast<__nv_bfloat16 *>(static_cast<char *>(packed) + sh.scale_off);
    const dim3 grid(sh.tiles, sh.groups);
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == G2_F32)
        q4_pack_kernel<float><<<grid, kPackThreads, 0, st>>>(static_cast<const float *>(W), transposed, codes, scales, sh);
    else
        q4_pack_kernel<__half><<<grid, kPackThreads, 0, st>>>(static_cast<const __half *>(W), transposed, codes, scales, sh);
    return launch_status(who);
}

extern "C" int g2k_q4_unpack(const void *packed, float *W, int N, int K, int group, void *stream) {
    const char *who = "g2k_q4_unpack";
    if (!W || !packed) return arg_error(G2_ERR_ARG, who, "null argument");
    int rc;
    if ((rc = check_packed(who, packed, N, K, group))) return rc;
    if ((rc = check_device_ptrs(who, {W, packed}))) return rc;
    const Q4Shape sh(N, K, group);
    const unsigned *codes = static_cast<const unsigned *>(packed);
    auto *scales = reinterpret_cast<const __nv_bfloat16 *>(static_cast<const char *>(packed) + sh.scale_off);
    const long long blocks = ((long long)K * N + 255) / 256;
    if (blocks > 0x7fffffffLL) return arg_error(G2_ERR_RANGE, who, "matrix too large");
    q4_unpack_kernel<<<(unsigned)blocks, 256, 0, (cudaStream_t)stream>>>(codes, scales, W, sh);
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
    Q4Args a{x, static_cast<const unsigned *>(packed),
             reinterpret_cast<const __nv_bfloat16 *>(static_cast<const char *>(packed) + sh.scale_off), bias, ln_gamma,
             ln_beta, residual, y, M, apply_gelu};
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == G2_F32)
        q4_matvec_kernel<float><<<(N + 7) / 8, 256, 0, st>>>(a, sh);
    else
        q4_matvec_kernel<__half><<<(N + 7) / 8, 256, 0, st>>>(a, sh);
    return launch_status(who);
}
