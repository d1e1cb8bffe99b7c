// g2_kv8.cu -- a paged KV cache of 8-bit codes with one scale for each page
// (block of tokens) and head: writing rows (g2k_kv8_append), reading them back
// (g2k_kv8_gather) and attention over it (g2k_kv8_attention).
//
// The value of a code c on a page with scale s is c s.  Codes are int8
// (-127..127) or e4m3 (up to 448).
#include <cuda_fp8.h>

#include <cmath>

#include "g2_args.h"
#include "g2_device.cuh"

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
    int first, n;   // rows of the sequence; n = 0: none, or out of range
};

__device__ __forceinline__ void bad(const Rows8 &r) {
    if (r.status) atomicExch(r.status, G2_ERR_RANGE);
}

__device__ __forceinline__ Span seq_rows(const Rows8 &r, int s) {
    Span p{s, 1};
    if (r.q_start) {
        p.first = r.q_start[s];
        const long long n = (long long)r.q_start[s + 1] - p.first;
        if (n < 0 || n > r.max_q || p.first < 0 || p.first + n > r.n_rows) {
            bad(r);
            return Span{0, 0};
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

// ---- append -----------------------------------------------------------------------
// One CTA for each (block of a sequence, head, K or V): the new rows' largest
// magnitude as an integer maximum (NaN above infinity above finite), the scale,
// the kept rows again if it grew, the new rows' codes.  A thread holds its
// 4-element vectors of the block in registers between the two passes.
constexpr int kAppendThreads = 256;

template <typename T, int FMT, int VPT>
__global__ void __launch_bounds__(kAppendThreads)
    kv8_append_kernel(g2_kv8 c, const T *k, const T *v, long long stride, const int *pos, Rows8 r, int blocks_per_seq) {
    __shared__ unsigned peaks[kAppendThreads / 32];
    const int t = threadIdx.x;
    const int s = blockIdx.x / blocks_per_seq, h = blockIdx.y, is_v = blockIdx.z;
    const int P = c.page_size, D = c.head_dim, per_row = D / 4;
    const Span sp = seq_rows(r, s);
    if (sp.n == 0) return;
    const int p0 = pos[s];
    if (p0 < 0 || (long long)p0 + sp.n > (long long)r.table_stride * P) {
        bad(r);
        return;
    }
    const int block = p0 / P + blockIdx.x % blocks_per_seq;
    const long long start = (long long)block * P;
    if (start >= (long long)p0 + sp.n) return;
    const int page = page_of(r, c, s, block);
    if (page < 0) return;
    const int kept = max(0, (int)(p0 - start));                        // rows 0..kept-1 stay
    const int end = (int)min((long long)P, (long long)p0 + sp.n - start);   // rows kept..end-1 are new
    const T *src = (is_v ? v : k) + (sp.first + start - p0) * stride + (long long)h * D;
    const long long at = (long long)page * c.n_kv_head + h;
    unsigned char *dst = static_cast<unsigned char *>(is_v ? c.v : c.k) + at * P * D;
    float *scale = (is_v ? c.v_scale : c.k_scale) + at;

    float4 x[VPT];
    unsigned peak = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int vec = t + i * kAppendThreads, row = vec / per_row;
        if (row >= kept && row < end) {
            x[i] = load4<T>(src + (long long)row * stride + (vec % per_row) * 4);
            peak = max(max(peak, max(abs_bits(x[i].x), abs_bits(x[i].y))), max(abs_bits(x[i].z), abs_bits(x[i].w)));
        }
    }
    const float was = kept > 0 ? *scale : 0.0f;
    peak = __reduce_max_sync(0xffffffffu, peak);
    if ((t & 31) == 0) peaks[t >> 5] = peak;
    __syncthreads();
    peak = peaks[0];
#pragma unroll
    for (int i = 1; i < kAppendThreads / 32; ++i) peak = max(peak, peaks[i]);
    float to = fmaxf(__fdiv_rn(__uint_as_float(peak), FMT == G2_KV_I8 ? 127.0f : 448.0f), kScaleFloor);
    if (peak >= 0x7f800000u || was != was) to = __uint_as_float(0x7fc00000u);
    else if (was > to) to = was;
    const bool again = to > was;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int vec = t + i * kAppendThreads, row = vec / per_row;
        unsigned *out = reinterpret_cast<unsigned *>(dst) + vec;
        if (row < kept) {
            if (again) {
                const unsigned w = *out;
                *out = recode<FMT>(w & 0xffu, was, to) | recode<FMT>((w >> 8) & 0xffu, was, to) << 8 |
                       recode<FMT>((w >> 16) & 0xffu, was, to) << 16 | recode<FMT>(w >> 24, was, to) << 24;
            }
        } else if (row < end) {
            unsigned w = 0;
            if (to == to)
                w = encode<FMT>(div_odd(x[i].x, to)) | encode<FMT>(div_odd(x[i].y, to)) << 8 |
                    encode<FMT>(div_odd(x[i].z, to)) << 16 | encode<FMT>(div_odd(x[i].w, to)) << 24;
            *out = w;
        }
    }
    if (t == 0) *scale = to;
}

// ---- gather -----------------------------------------------------------------------
constexpr int kGatherRows = 16;

template <typename T, int FMT>
__global__ void __launch_bounds__(256)
    kv8_gather_kernel(g2_kv8 c, T *k, T *v, long long stride, const int *pos, Rows8 r, int groups_per_seq) {
    const int s = blockIdx.x / groups_per_seq, h = blockIdx.y;
    const int P = c.page_size, D = c.head_dim, per_row = D / 4;
    const Span sp = seq_rows(r, s);
    if (sp.n == 0) return;
    const int p0 = pos[s];
    if (p0 < 0 || (long long)p0 + sp.n > (long long)r.table_stride * P) {
        bad(r);
        return;
    }
    const int j0 = blockIdx.x % groups_per_seq * kGatherRows, j1 = min(sp.n, j0 + kGatherRows);
    for (int i = threadIdx.x; i < (j1 - j0) * per_row * 2; i += 256) {
        const int is_v = i >= (j1 - j0) * per_row, q = is_v ? i - (j1 - j0) * per_row : i;
        const int j = j0 + q / per_row, d = q % per_row * 4, p = p0 + j;
        const int page = page_of(r, c, s, p / P);
        if (page < 0) continue;
        const long long at = (long long)page * c.n_kv_head + h;
        const unsigned w = *reinterpret_cast<const unsigned *>(static_cast<const unsigned char *>(is_v ? c.v : c.k) +
                                                               (at * P + p % P) * D + d);
        const float sc = (is_v ? c.v_scale : c.k_scale)[at];
        T *o = (is_v ? v : k) + (sp.first + j) * stride + (long long)h * D + d;
        o[0] = fromf<T>(decode<FMT>(w & 0xffu) * sc);
        o[1] = fromf<T>(decode<FMT>((w >> 8) & 0xffu) * sc);
        o[2] = fromf<T>(decode<FMT>((w >> 16) & 0xffu) * sc);
        o[3] = fromf<T>(decode<FMT>(w >> 24) * sc);
    }
}

// ---- attention --------------------------------------------------------------------
// One CTA for each query row and head, keys in tiles of 128: a key per thread
// for the scores, a dimension per thread for the sums, with the running
// maximum and sum of the softmax carried from tile to tile.
constexpr int kAttnThreads = 128;

template <typename T, int FMT>
__global__ void __launch_bounds__(kAttnThreads)
    kv8_attention_kernel(g2_kv8 c, const T *q, long long q_stride, T *out, long long out_stride, int group, float scale,
                         const int *seq_len, Rows8 r) {
    __shared__ float qs[128], ps[kAttnThreads], red[kAttnThreads / 32];
    __shared__ int pages[kAttnThreads];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int s = blockIdx.x / r.max_q, j = blockIdx.x % r.max_q, h = blockIdx.y, kh = h / group;
    const int P = c.page_size, D = c.head_dim;
    const Span sp = seq_rows(r, s);
    if (j >= sp.n) return;
    const int len = seq_len[s];
    if (len < 0 || len > (long long)r.table_stride * P) {
        bad(r);
        return;
    }
    const int keys = len - sp.n + j + 1;
    const long long row = sp.first + j;
    if (t < D) qs[t] = tof(q[row * q_stride + (long long)h * D + t]) * scale;
    float m = -INFINITY, l = 0.0f, acc = 0.0f;
    for (int k0 = 0; k0 < keys; k0 += kAttnThreads) {
        __syncthreads();
        const int key = k0 + t;
        float sc = -INFINITY;
        pages[t] = -1;
        if (key < keys) {
            const int page = page_of(r, c, s, key / P);
            pages[t] = page;
            if (page >= 0) {
                const long long at = (long long)page * c.n_kv_head + kh;
                const unsigned char *p = static_cast<const unsigned char *>(c.k) + (at * P + key % P) * D;
                float dot = 0.0f;
                for (int d = 0; d < D; d += 4) {
                    const unsigned w = *reinterpret_cast<const unsigned *>(p + d);
                    dot += qs[d] * decode<FMT>(w & 0xffu) + qs[d + 1] * decode<FMT>((w >> 8) & 0xffu) +
                           qs[d + 2] * decode<FMT>((w >> 16) & 0xffu) + qs[d + 3] * decode<FMT>(w >> 24);
                }
                sc = dot * c.k_scale[at];
            }
        }
        float mx = sc;
        for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        if (lane == 0) red[warp] = mx;
        __syncthreads();
        mx = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
        const float base = mx == -INFINITY ? 0.0f : mx;
        const float p = expf(sc - base), fix = expf(m - base);
        ps[t] = p;
        __syncthreads();
        float sum = 0.0f;
        acc *= fix;
        const int n = min(kAttnThreads, keys - k0);
        for (int i = 0; i < n; ++i) {
            sum += ps[i];
            if (t < D && pages[i] >= 0) {
                const long long at = (long long)pages[i] * c.n_kv_head + kh;
                acc += ps[i] * decode<FMT>(static_cast<const unsigned char *>(c.v)[(at * P + (k0 + i) % P) * D + t]) * c.v_scale[at];
            }
        }
        l = l * fix + sum;
        m = mx;
    }
    if (t < D) out[row * out_stride + (long long)h * D + t] = fromf<T>(l > 0.0f || l != l ? acc / l : 0.0f);
}

// ---- argument checks ----------------------------------------------------------------
int check_cache(const char *who, const g2_kv8 *c) {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) return arg_error(G2_ERR_ARG, who, "null cache or cache array");
    if (c->format != G2_KV_I8 && c->format != G2_KV_E4M3) return arg_error(G2_ERR_ARG, who, "bad cache format");
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
        return arg_error(G2_ERR_ARG, who, "page_size must be 16, 32, 64 or 128");
    if (c->head_dim != 64 && c->head_dim != 128) return arg_error(G2_ERR_ARG, who, "head_dim must be 64 or 128");
    if (c->n_pages < 1 || c->n_kv_head < 1 || c->n_kv_head > 65535)
        return arg_error(G2_ERR_RANGE, who, "need n_pages >= 1 and 1 <= n_kv_head <= 65535");
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
    if ((long long)r.table_stride * c->page_size > 0x7fffffffLL)
        return arg_error(G2_ERR_RANGE, who, "a table row holds more than 2^31 - 1 positions");
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
void launch_append(const g2_kv8 &c, const void *k, const void *v, long long stride, const int *pos, const Rows8 &r,
                   cudaStream_t st) {
    const int per = (c.page_size - 1 + r.max_q - 1) / c.page_size + 1;   // blocks that max_q rows can touch
    const dim3 grid((unsigned)per * r.n_seq, c.n_kv_head, 2);
    const T *kt = static_cast<const T *>(k), *vt = static_cast<const T *>(v);
    switch (c.page_size * c.head_dim / (4 * kAppendThreads)) {
        case 1: kv8_append_kernel<T, FMT, 1><<<grid, kAppendThreads, 0, st>>>(c, kt, vt, stride, pos, r, per); break;
        case 2: kv8_append_kernel<T, FMT, 2><<<grid, kAppendThreads, 0, st>>>(c, kt, vt, stride, pos, r, per); break;
        case 4: kv8_append_kernel<T, FMT, 4><<<grid, kAppendThreads, 0, st>>>(c, kt, vt, stride, pos, r, per); break;
        case 8: kv8_append_kernel<T, FMT, 8><<<grid, kAppendThreads, 0, st>>>(c, kt, vt, stride, pos, r, per); break;
        default: kv8_append_kernel<T, FMT, 16><<<grid, kAppendThreads, 0, st>>>(c, kt, vt, stride, pos, r, per); break;
    }
}

template <typename T, int FMT>
void launch_gather(const g2_kv8 &c, void *k, void *v, long long stride, const int *pos, const Rows8 &r, cudaStream_t st) {
    const int per = (r.max_q + kGatherRows - 1) / kGatherRows;
    kv8_gather_kernel<T, FMT><<<dim3((unsigned)per * r.n_seq, c.n_kv_head), 256, 0, st>>>(
        c, static_cast<T *>(k), static_cast<T *>(v), stride, pos, r, per);
}

template <typename T, int FMT>
void launch_attention8(const g2_kv8 &c, const void *q, long long q_stride, void *out, long long out_stride, int n_head,
                       float scale, const int *seq_len, const Rows8 &r, cudaStream_t st) {
    kv8_attention_kernel<T, FMT><<<dim3((unsigned)r.max_q * r.n_seq, n_head), kAttnThreads, 0, st>>>(
        c, static_cast<const T *>(q), q_stride, static_cast<T *>(out), out_stride, n_head / c.n_kv_head, scale, seq_len, r);
}

// dtype and format to template arguments
#define G2_KV8_DISPATCH(fn, ...)                                     \
    do {                                                             \
        if (dtype == G2_F32 && cache->format == G2_KV_I8)            \
            fn<float, G2_KV_I8>(__VA_ARGS__);                        \
        else if (dtype == G2_F32)                                    \
            fn<float, G2_KV_E4M3>(__VA_ARGS__);                      \
        else if (cache->format == G2_KV_I8)                          \
            fn<__half, G2_KV_I8>(__VA_ARGS__);                       \
        else                                                         \
            fn<__half, G2_KV_E4M3>(__VA_ARGS__);                     \
    } while (0)

}  // namespace

}  // namespace g2

using namespace g2;

extern "C" int g2k_kv8_append(const g2_kv8 *cache, const void *k, const void *v, int dtype, long long row_stride, int n_rows,
                              int n_seq, const int *q_start, const int *pos, int max_q, const int *table, int table_stride,
                              int *status, void *stream) {
    const char *who = "g2k_kv8_append";
    int rc;
    if ((rc = check_cache(who, cache))) return rc;
    const Rows8 r{n_rows, n_seq, max_q, q_start, table, table_stride, status};
    if ((rc = check_rows(who, cache, cache->n_kv_head, k, v, dtype, &row_stride, nullptr, r, pos))) return rc;
    if (((long long)max_q / cache->page_size + 2) * n_seq > 0x7fffffffLL) return arg_error(G2_ERR_RANGE, who, "too many blocks");
    if (n_rows == 0 || n_seq == 0) return G2_OK;
    if ((rc = check_device_ptrs(who, {cache->k, cache->v, cache->k_scale, cache->v_scale, k, v, q_start, pos, table, status})))
        return rc;
    G2_KV8_DISPATCH(launch_append, *cache, k, v, row_stride, pos, r, (cudaStream_t)stream);
    return launch_status(who);
}

extern "C" int g2k_kv8_gather(const g2_kv8 *cache, void *k_out, void *v_out, int dtype, long long row_stride, int n_rows,
                              int n_seq, const int *q_start, const int *pos, int max_q, const int *table, int table_stride,
                              int *status, void *stream) {
    const char *who = "g2k_kv8_gather";
    int rc;
    if ((rc = check_cache(who, cache))) return rc;
    const Rows8 r{n_rows, n_seq, max_q, q_start, table, table_stride, status};
    if ((rc = check_rows(who, cache, cache->n_kv_head, k_out, v_out, dtype, &row_stride, nullptr, r, pos))) return rc;
    if (((long long)max_q / kGatherRows + 1) * n_seq > 0x7fffffffLL) return arg_error(G2_ERR_RANGE, who, "too many rows");
    if (n_rows == 0 || n_seq == 0) return G2_OK;
    if ((rc = check_device_ptrs(who, {cache->k, cache->v, cache->k_scale, cache->v_scale, k_out, v_out, q_start, pos, table, status})))
        return rc;
    G2_KV8_DISPATCH(launch_gather, *cache, k_out, v_out, row_stride, pos, r, (cudaStream_t)stream);
    return launch_status(who);
}

extern "C" size_t g2k_kv8_attention_workspace(const g2_kv8 *cache, int n_head, int n_seq, int max_q) {
    if (!cache || n_head < 1 || n_seq < 0 || max_q < 1) return 0;
    return 256;
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
    if (!(scale > 0.0f) || !std::isfinite(scale)) return arg_error(G2_ERR_ARG, who, "scale must be positive");
    const Rows8 r{n_rows, n_seq, max_q, q_start, table, table_stride, status};
    if ((rc = check_rows(who, cache, n_head, q, out, dtype, &q_stride, &out_stride, r, seq_len))) return rc;
    if ((long long)max_q * n_seq > 0x7fffffffLL) return arg_error(G2_ERR_RANGE, who, "too many rows");
    if (!workspace || !aligned(workspace, 256)) return arg_error(G2_ERR_ARG, who, "workspace not 256-byte aligned");
    if (workspace_bytes < g2k_kv8_attention_workspace(cache, n_head, n_seq, max_q))
        return arg_error(G2_ERR_ARG, who, "workspace too small");
    if (n_rows == 0 || n_seq == 0) return G2_OK;
    if ((rc = check_device_ptrs(who, {cache->k, cache->v, cache->k_scale, cache->v_scale, q, out, q_start, seq_len, table,
                                      workspace, status})))
        return rc;
    G2_KV8_DISPATCH(launch_attention8, *cache, q, q_stride, out, out_stride, n_head, scale, seq_len, r, (cudaStream_t)stream);
    return launch_status(who);
}
