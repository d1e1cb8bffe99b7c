// g2_logits.cu -- rules on rows of logits before a token is picked: penalties
// for tokens of the context, biases and grammar masks (g2k_process_logits).
//
// One CTA for each slice of kSlice columns of a row.
//   1. The columns are copied, masked ones as G2_MASKED, four at a time (slices
//      begin where a row's address is a multiple of 16 bytes, whatever the stride).
//      In place only masked columns are written and nothing is read.
//   2. Meanwhile the context's ids that fall into the slice are counted in shared
//      memory (integer additions, so their order does not matter), and each biased
//      column notes the last pair that names it.  Whoever touches a column first
//      puts it on a list.
//   3. The columns of the list are computed and written over the copy: a context
//      touches about one column in a hundred, and testing all of them in the copy
//      took longer than the copy (256 rows of 50257: 37 us).
// The context and the pairs are read by every slice of the row, from L2 after the
// first.  Bound by the bytes of the logits, read and written once.
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

constexpr unsigned kSeen = 0x80000000u, kBiased = 0x40000000u, kCount = 0x3fffffffu;

template <bool PENAL, bool BIAS, bool MASK>
__global__ void __launch_bounds__(kRuleThreads) rules_kernel(RuleArgs a) {
    constexpr bool SPARSE = PENAL || BIAS;
    __shared__ __align__(16) unsigned count[SPARSE ? kSlice : 4];   // ids after the prompt, and kSeen / kBiased
    __shared__ int pair[BIAS ? kSlice : 1];                         // last pair of a biased column
    __shared__ unsigned short list[SPARSE ? kSlice : 1];            // touched columns
    __shared__ unsigned n_list;
    const int t = threadIdx.x, row = blockIdx.y;
    const g2_logit_rules &r = a.r;
    const float *in = a.logits + row * a.ld;
    float *out = a.out + row * a.ld_out;
    const bool in_place = in == out;
    const int shift = (int)(reinterpret_cast<size_t>(out) / 4 & 3);
    const bool same = (int)(reinterpret_cast<size_t>(in) / 4 & 3) == shift;
    const int v0 = blockIdx.x * kSlice - shift;                     // below 0 in the first slice
    if (v0 >= a.V) return;                                          // the last slice of a row without a shift
    const unsigned *mask = MASK ? r.mask + (long long)row * r.mask_stride : nullptr;

    // ---- requests of the copy
    float4 l[kVecs];
    unsigned allowed[kVecs];
    auto column = [&](int i) { return v0 + 4 * (t + i * kRuleThreads); };
    auto whole = [&](int c) { return c >= 0 && c + 3 < a.V; };
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int c = column(i);
        if (!in_place) {
            if (same && whole(c)) {
                l[i] = __ldcs(reinterpret_cast<const float4 *>(in + c));
            } else {
                float *e = &l[i].x;
#pragma unroll
                for (int j = 0; j < 4; ++j) e[j] = c + j >= 0 && c + j < a.V ? in[c + j] : 0.0f;
            }
        }
        if (MASK) {
            const int w0 = max(c, 0) >> 5, w1 = min(max(c, 0) + 3, a.V - 1) >> 5;
            const unsigned lo = c < a.V ? mask[w0] : 0u, hi = c < a.V ? mask[w1] : 0u;
            // bits c .. c + 3; a first group that begins before column 0 has its bits moved up
            allowed[i] = c >= 0 ? __funnelshift_r(lo, hi, c & 31) : lo << -c;
        }
    }
    // ---- the tables
    int c0 = 0, c1 = 0, b0 = 0, b1 = 0;
    long long made = 0;
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    if (SPARSE) {
        for (int i = t; i < kSlice / 4; i += kRuleThreads) reinterpret_cast<uint4 *>(count)[i] = make_uint4(0, 0, 0, 0);
        if (t == 0) n_list = 0;
    }
    if (BIAS)
        for (int i = t; i < kSlice; i += kRuleThreads) pair[i] = -1;
    if (PENAL) {
        span_of(r.ctx_start, row, r.n_ctx, c0, c1);
        made = (long long)c0 + (r.n_prompt ? max(r.n_prompt[row], 0) : 0);
        if (r.rep_penalty) rep = r.rep_penalty[row];
        if (r.frequency) freq = r.frequency[row];
        if (r.presence) pres = r.presence[row];
        if (!(rep > 0.0f)) rep = 1.0f;
    }
    if (BIAS) span_of(r.bias_start, row, r.n_bias, b0, b1);
    if (SPARSE) __syncthreads();
    const unsigned n = min(kSlice, a.V - v0);
    auto touched = [&](unsigned at, unsigned old) {
        if (old == 0) list[atomicAdd(&n_list, 1u)] = (unsigned short)at;
    };
    if (PENAL) {
#pragma unroll 4
        for (int i = c0 + t; i < c1; i += kRuleThreads) {
            const int id = r.ctx[i];
            const unsigned at = (unsigned)(id - v0);
            if (id >= 0 && at < n) {
                touched(at, atomicOr(&count[at], kSeen));
                if (i >= made) atomicAdd(&count[at], 1u);
            }
        }
    }
    if (BIAS) {
#pragma unroll 4
        for (int i = b0 + t; i < b1; i += kRuleThreads) {
            const int id = r.bias_ids[i];
            const unsigned at = (unsigned)(id - v0);
            if (id >= 0 && at < n) {
                touched(at, atomicOr(&count[at], kBiased));
                atomicMax(&pair[at], i);
            }
        }
    }
    // ---- the copy
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int c = column(i);
        if (c >= a.V) break;
        float *e = &l[i].x;
        const unsigned ok = MASK ? allowed[i] & 15u : 15u;
        if (in_place && ok == 15u) continue;
        if (MASK) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (!((ok >> j) & 1u)) e[j] = G2_MASKED;
        }
        if (whole(c) && (!in_place || ok == 0)) {
            __stcs(reinterpret_cast<float4 *>(out + c), l[i]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c + j >= 0 && c + j < a.V && (!in_place || !((ok >> j) & 1u))) out[c + j] = e[j];
        }
    }
    if (!SPARSE) return;
    __syncthreads();
    // ---- the touched columns, after their copies
    for (unsigned i = t; i < n_list; i += kRuleThreads) {
        const int at = list[i], c = v0 + at;
        if (MASK && !((mask[c >> 5] >> (c & 31)) & 1u)) continue;
        const unsigned q = count[at];
        float x = in[c];
        if (PENAL && (q & kSeen)) {
            x = x > 0.0f ? x / rep : x * rep;
            if (q & kCount) {
                x -= freq * (float)(q & kCount);
                x -= pres;
            }
        }
        if (BIAS && (q & kBiased)) x += r.bias[pair[at]];
        out[c] = x;
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
