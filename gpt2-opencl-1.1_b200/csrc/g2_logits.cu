// g2_logits.cu -- rules on rows of logits before a token is picked: penalties
// for tokens of the context, biases and grammar masks (g2k_process_logits).
//
// One CTA for each slice of kSlice columns of a row.  It counts the context's
// ids that fall into its slice in shared memory (integer additions, so their
// order does not matter), notes for each biased column the last pair that names
// it, and passes over its columns once.  The context and the pairs are read by
// every slice of the row, from L2 after the first.
#include "g2_args.h"
#include "g2_device.cuh"

namespace g2 {

namespace {

constexpr int kSlice = 4096, kRuleThreads = 256;

struct RuleArgs {
    const float *logits;
    float *out;
    long long ld, ld_out;
    int V;
    g2_logit_rules r;
};

// clamps [start, end) to [0, n)
__device__ __forceinline__ void span_of(const int *start, int row, int n, int &a, int &b) {
    a = start ? min(max(start[row], 0), n) : 0;
    b = start ? min(max(start[row + 1], a), n) : n;
}

__global__ void __launch_bounds__(kRuleThreads) rules_kernel(RuleArgs a) {
    __shared__ unsigned count[kSlice];   // ids after the prompt; top bit: anywhere in the context
    __shared__ int pair[kSlice];         // last pair of the column + 1
    const int t = threadIdx.x, row = blockIdx.y;
    const int v0 = blockIdx.x * kSlice, n = min(kSlice, a.V - v0);
    const g2_logit_rules &r = a.r;
    const bool penal = r.ctx && (r.rep_penalty || r.presence || r.frequency);
    if (penal)
        for (int i = t; i < n; i += kRuleThreads) count[i] = 0;
    if (r.bias_ids)
        for (int i = t; i < n; i += kRuleThreads) pair[i] = 0;
    __syncthreads();
    if (penal) {
        int c0, c1;
        span_of(r.ctx_start, row, r.n_ctx, c0, c1);
        const long long made = (long long)c0 + (r.n_prompt ? max(r.n_prompt[row], 0) : 0);
        for (int i = c0 + t; i < c1; i += kRuleThreads) {
            const unsigned at = (unsigned)(r.ctx[i] - v0);
            if (at < (unsigned)n) {
                if (i >= made) atomicAdd(&count[at], 1u);
                atomicOr(&count[at], 0x80000000u);
            }
        }
    }
    if (r.bias_ids) {
        int b0, b1;
        span_of(r.bias_start, row, r.n_bias, b0, b1);
        for (int i = b0 + t; i < b1; i += kRuleThreads) {
            const unsigned at = (unsigned)(r.bias_ids[i] - v0);
            if (at < (unsigned)n) atomicMax(&pair[at], i + 1);
        }
    }
    __syncthreads();
    float rep = r.rep_penalty ? r.rep_penalty[row] : 1.0f;
    if (!(rep > 0.0f)) rep = 1.0f;
    const float freq = r.frequency ? r.frequency[row] : 0.0f, pres = r.presence ? r.presence[row] : 0.0f;
    const unsigned *mask = r.mask ? r.mask + (long long)row * r.mask_stride : nullptr;
    const float *in = a.logits + row * a.ld + v0;
    float *out = a.out + row * a.ld_out + v0;
    for (int i = t; i < n; i += kRuleThreads) {
        float l = in[i];
        if (penal && count[i]) {
            l = l > 0.0f ? l / rep : l * rep;
            const unsigned c = count[i] & 0x7fffffffu;
            if (c) {
                l -= freq * (float)c;
                l -= pres;
            }
        }
        if (r.bias_ids && pair[i]) l += r.bias[pair[i] - 1];
        if (mask && !((mask[(v0 + i) >> 5] >> ((v0 + i) & 31)) & 1u)) l = G2_MASKED;
        out[i] = l;
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
    RuleArgs a{logits, out, ld, ld_out, vocab, rules};
    if (rules.n_ctx == 0) a.r.ctx = nullptr;
    if (rules.n_bias == 0) a.r.bias_ids = nullptr;
    rules_kernel<<<dim3((vocab + kSlice - 1) / kSlice, rows), kRuleThreads, 0, st>>>(a);
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
