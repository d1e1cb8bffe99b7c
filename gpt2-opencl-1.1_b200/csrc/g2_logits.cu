// g2_logits.cu -- rules on rows of logits before a token is picked: penalties
// for tokens of the context, biases and grammar masks (g2k_process_logits).
//
// One CTA for each slice of kSlice columns of a row.  It requests its logits and
// mask words, then counts the context's ids that fall into its slice in shared
// memory (integer additions, so their order does not matter) and notes for each
// biased column the last pair that names it, and so passes over its columns once,
// with the tables built while the logits are on their way.  The context and the
// pairs are read by every slice of the row, from L2 after the first.  Bound by the
// bytes of the logits, read and written once.  Slices begin where a row's address
// is a multiple of 16 bytes, whatever the row stride, so that four columns move at
// a time.
#include "g2_args.h"
#include "g2_device.cuh"

namespace g2 {

namespace {

constexpr int kSlice = 4096, kRuleThreads = 256, kVecs = kSlice / 4 / kRuleThreads;

struct RuleArgs {
    const float *logits;
    float *out;
    long long ld, ld_out;
    int V;
    g2_logit_rules r;
};

// clamps [start, end) to [0, n)
__device__ __forceinline__ void span_of(const int *start, int row, int n, int &a, int &b) {
    a = 0;
    b = n;
    if (start) {
        const int s0 = start[row], s1 = start[row + 1];
        a = min(max(s0, 0), n);
        b = min(max(s1, a), n);
    }
}

template <bool PENAL, bool BIAS, bool MASK>
__global__ void __launch_bounds__(kRuleThreads) rules_kernel(RuleArgs a) {
    __shared__ __align__(16) unsigned count[PENAL ? kSlice : 4];   // ids after the prompt; top bit: anywhere in the context
    __shared__ __align__(16) int pair[BIAS ? kSlice : 4];          // last pair of the column + 1
    const int t = threadIdx.x, row = blockIdx.y;
    const g2_logit_rules &r = a.r;
    const float *in = a.logits + row * a.ld;
    float *out = a.out + row * a.ld_out;
    const int shift = (int)(reinterpret_cast<size_t>(in) / 4 & 3);
    const bool same = (int)(reinterpret_cast<size_t>(out) / 4 & 3) == shift, in_place = in == out;
    const int v0 = blockIdx.x * kSlice - shift;                    // below 0 in the first slice
    if (v0 >= a.V) return;                                         // the last slice of a row without a shift

    float4 l[kVecs];
    unsigned allowed[kVecs];
    auto column = [&](int i) { return v0 + 4 * (t + i * kRuleThreads); };
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int c = column(i);
        if (c >= 0 && c + 3 < a.V) {
            l[i] = __ldcs(reinterpret_cast<const float4 *>(in + c));
        } else {
            float *e = &l[i].x;
#pragma unroll
            for (int j = 0; j < 4; ++j) e[j] = c + j >= 0 && c + j < a.V ? in[c + j] : 0.0f;
        }
        if (MASK) {
            const unsigned *mask = r.mask + (long long)row * r.mask_stride;
            const int w0 = max(c, 0) >> 5, w1 = min(max(c, 0) + 3, a.V - 1) >> 5;
            const unsigned lo = c < a.V ? mask[w0] : 0u, hi = c < a.V ? mask[w1] : 0u;
            // bits c .. c + 3; a first group that begins before column 0 has its bits moved up
            allowed[i] = c >= 0 ? __funnelshift_r(lo, hi, c & 31) : lo << -c;
        }
    }
    if (PENAL)
        for (int i = t; i < kSlice / 4; i += kRuleThreads) reinterpret_cast<uint4 *>(count)[i] = make_uint4(0, 0, 0, 0);
    if (BIAS)
        for (int i = t; i < kSlice / 4; i += kRuleThreads) reinterpret_cast<uint4 *>(pair)[i] = make_uint4(0, 0, 0, 0);
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    if (PENAL) {
        if (r.rep_penalty) rep = r.rep_penalty[row];
        if (r.frequency) freq = r.frequency[row];
        if (r.presence) pres = r.presence[row];
        if (!(rep > 0.0f)) rep = 1.0f;
    }
    if (PENAL || BIAS) __syncthreads();
    const int n = min(kSlice, a.V - v0);
    if (PENAL) {
        int c0, c1;
        span_of(r.ctx_start, row, r.n_ctx, c0, c1);
        const long long made = (long long)c0 + (r.n_prompt ? max(r.n_prompt[row], 0) : 0);
#pragma unroll 4
        for (int i = c0 + t; i < c1; i += kRuleThreads) {
            const int id = r.ctx[i];
            const unsigned at = (unsigned)(id - v0);
            if (id >= 0 && at < (unsigned)n) {
                if (i >= made) atomicAdd(&count[at], 1u);
                atomicOr(&count[at], 0x80000000u);
            }
        }
    }
    if (BIAS) {
        int b0, b1;
        span_of(r.bias_start, row, r.n_bias, b0, b1);
#pragma unroll 4
        for (int i = b0 + t; i < b1; i += kRuleThreads) {
            const int id = r.bias_ids[i];
            const unsigned at = (unsigned)(id - v0);
            if (id >= 0 && at < (unsigned)n) atomicMax(&pair[at], i + 1);
        }
    }
    if (PENAL || BIAS) __syncthreads();
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int c = column(i);
        if (c >= a.V) break;
        float *e = &l[i].x;
        bool changed = !in_place;
        if (PENAL) {
            const uint4 q = reinterpret_cast<const uint4 *>(count)[t + i * kRuleThreads];
            if (q.x | q.y | q.z | q.w) {
                changed = true;
                const unsigned cs[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (cs[j]) {
                        e[j] = e[j] > 0.0f ? e[j] / rep : e[j] * rep;
                        const unsigned k = cs[j] & 0x7fffffffu;
                        if (k) {
                            e[j] -= freq * (float)k;
                            e[j] -= pres;
                        }
                    }
            }
        }
        if (BIAS) {
            const int4 q = reinterpret_cast<const int4 *>(pair)[t + i * kRuleThreads];
            if (q.x | q.y | q.z | q.w) {
                changed = true;
                const int ps[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (ps[j]) e[j] += r.bias[ps[j] - 1];
            }
        }
        if (MASK && (allowed[i] & 15u) != 15u) {
            changed = true;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (!((allowed[i] >> j) & 1u)) e[j] = G2_MASKED;
        }
        if (!changed) continue;
        if (same && c >= 0 && c + 3 < a.V) {
            __stcs(reinterpret_cast<float4 *>(out + c), l[i]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c + j >= 0 && c + j < a.V) out[c + j] = e[j];
        }
    }
}

}  // namespace

// Host checks of the rules; `device`: arrays of `rows` rows in device memory, else host arrays of one.
int check_rules(const char *who, const g2_logit_rules *r, int rows, int vocab, bool device) {
    if (!r) return arg_error(G2_ERR_ARG, who, "null rules");
    if (r->n_ctx < 0 || r->n_bias < 0 || r->mask_stride < 0)
        return arg_error(G2_ERR_RANGE, who, "need n_ctx >= 0, n_bias >= 0 and mask_stride >= 0");
    if (r->n_ctx > 0 && !r->ctx) return arg_error(G2_ERR_ARG, who, "n_ctx without ctx");
    if (r->n_bias > 0 && (!r->bias_ids || !r->bias)) return arg_error(G2_ERR_ARG, who, "n_bias without bias_ids and bias");
    if (device && rows > 1 && ((r->n_ctx > 0 && !r->ctx_start) || (r->n_bias > 0 && !r->bias_start)))
        return arg_error(G2_ERR_ARG, who, "several rows need ctx_start and bias_start");
    if (r->mask && r->mask_stride && r->mask_stride < (vocab + 31) / 32)
        return arg_error(G2_ERR_RANGE, who, "mask_stride is less than a row of the mask");
    for (const void *p : {(const void *)r->ctx, (const void *)r->ctx_start, (const void *)r->n_prompt,
                          (const void *)r->rep_penalty, (const void *)r->presence, (const void *)r->frequency,
                          (const void *)r->bias_ids, (const void *)r->bias, (const void *)r->bias_start, (const void *)r->mask})
        if (!aligned(p, 4)) return arg_error(G2_ERR_ARG, who, "an array is not 4-byte aligned");
    return G2_OK;
}

void launch_rules(const float *logits, long long ld, float *out, long long ld_out, int rows, int vocab,
                  const g2_logit_rules &rules, cudaStream_t st) {
    const RuleArgs a{logits, out, ld, ld_out, vocab, rules};
    const dim3 grid((vocab + 3 + kSlice - 1) / kSlice, rows);   // 3: a row that begins past a multiple of 16 bytes
    const bool penal = rules.n_ctx > 0 && (rules.rep_penalty || rules.presence || rules.frequency), bias = rules.n_bias > 0;
    void (*const kernels[8])(RuleArgs) = {
        rules_kernel<false, false, false>, rules_kernel<true, false, false>, rules_kernel<false, true, false>, rules_kernel<true, true, false>,
        rules_kernel<false, false, true>,  rules_kernel<true, false, true>,  rules_kernel<false, true, true>,  rules_kernel<true, true, true>};
    kernels[(penal ? 1 : 0) + (bias ? 2 : 0) + (rules.mask ? 4 : 0)]<<<grid, kRuleThreads, 0, st>>>(a);
}

}  // namespace g2

using namespace g2;

extern "C" int g2k_process_logits(const float *logits, long long ld, float *out, long long ld_out, int rows, int vocab_size,
                                  const g2_logit_rules *rules, void *stream) {
    const char *who = "g2k_process_logits";
    if (!logits || !out) return arg_error(G2_ERR_ARG, who, "null argument");
    if (rows < 0 || rows > 65535 || vocab_size < 1)
        return arg_error(G2_ERR_RANGE, who, "need 0 <= rows <= 65535 and vocab_size >= 1");
    if (rows > 1 && (ld < vocab_size || ld_out < vocab_size))
        return arg_error(G2_ERR_RANGE, who, "ld and ld_out must be at least vocab_size");
    if (out == logits && ld != ld_out && rows > 1) return arg_error(G2_ERR_ARG, who, "in place, ld and ld_out are the same");
    if (!aligned(logits, 4) || !aligned(out, 4)) return arg_error(G2_ERR_ARG, who, "logits are not 4-byte aligned");
    int rc;
    if ((rc = check_rules(who, rules, rows, vocab_size, true))) return rc;
    if (rows == 0) return G2_OK;
    if ((rc = check_device_ptrs(who, {logits, out, rules->ctx, rules->ctx_start, rules->n_prompt, rules->rep_penalty,
                                      rules->presence, rules->frequency, rules->bias_ids, rules->bias, rules->bias_start,
                                      rules->mask})))
        return rc;
    launch_rules(logits, ld, out, ld_out, rows, vocab_size, *rules, (cudaStream_t)stream);
    return launch_status(who);
}
