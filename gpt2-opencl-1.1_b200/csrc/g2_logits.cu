// g2_logits.cu -- rules on rows of logits before a token is picked: penalties
// for tokens of the context, biases and grammar masks (g2k_process_logits).
//
// One CTA for each slice of a row's columns; half of its warps begin with the copy
// (3) while the others build the tables (1, 2) and then join them.
//   1. The context's ids and the pairs' that fall into the slice set bits of a map
//      in shared memory; the bits before a column number the touched columns, so
//      that counts and pairs need memory for those only (kTouched at a time).
//   2. Counts by integer additions, whose order does not matter; of a column's pairs
//      the last by a maximum.
//   3. The slice's columns are copied, masked ones as G2_MASKED, four at a time
//      (slices begin where a row's address is a multiple of 16 bytes, whatever the
//      stride).  In place only masked columns are written and nothing is read.
//   4. The touched columns are computed and written over the copy.  A context touches
//      about one column in a hundred; testing all of them in the copy took longer
//      than the copy.
// Bound by the bytes of the logits, read and written once, and by what each CTA does
// before its copy is all on its way.  Rows are cut into about eight slices for each
// SM, of which five run at a time (256 threads of 48 registers): every slice of a row
// reads the whole context, and with slices of 4096 columns that took longer than the
// columns (256 rows of 50257: 37 us).
#include <algorithm>

#include "g2_args.h"
#include "g2_device.cuh"

namespace g2 {

namespace {

constexpr int kRuleThreads = 256, kTableThreads = 128;
constexpr int kVecs = 4, kStep = kVecs * 128;     // groups of four columns that a lane, columns that a warp copies at a time
constexpr int kTouched = 2048;
constexpr int kMinSlice = 4096, kMaxSlice = 65536;

struct RuleArgs {
    const float *logits;
    float *out;
    long long ld, ld_out;
    int V, slice;
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

constexpr unsigned kSeen = 0x80000000u, kCount = 0x7fffffffu;

template <bool PENAL, bool BIAS, bool MASK>
__global__ void __launch_bounds__(kRuleThreads) rules_kernel(RuleArgs a) {
    constexpr bool SPARSE = PENAL || BIAS;
    extern __shared__ unsigned map[];                        // [slice / 32] bits of touched columns, then as many counts of bits before
    __shared__ unsigned count[PENAL ? kTouched : 1];         // ids after the prompt, and kSeen
    __shared__ int pair[BIAS ? kTouched : 1];                // last pair, or -1
    __shared__ int list[SPARSE ? kTouched : 1];              // columns
    __shared__ unsigned warp_sum[kTableThreads / 32];
    __shared__ unsigned touched_s;                           // touched columns
    __shared__ int next;                                     // step of the copy
    const int t = threadIdx.x, lane = t & 31, row = blockIdx.y;
    const g2_logit_rules &r = a.r;
    pdl_wait();
    pdl_launch();
    const float *in = a.logits + row * a.ld;
    float *out = a.out + row * a.ld_out;
    const bool in_place = in == out;
    const int shift = (int)(reinterpret_cast<size_t>(out) / 4 & 3);
    const bool same = (int)(reinterpret_cast<size_t>(in) / 4 & 3) == shift;
    const int v0 = blockIdx.x * a.slice - shift;             // below 0 in the first slice
    if (v0 >= a.V) return;                                   // the last slice of a row without a shift
    const int n = min(a.slice, a.V - v0);                    // columns v0 .. v0 + n - 1
    const unsigned *mask = MASK ? r.mask + (long long)row * r.mask_stride : nullptr;
    const int words = a.slice / 32;
    unsigned *before = map + words;

    // ---- the tables, by the first kTableThreads threads
    auto table_sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(kTableThreads) : "memory"); };
    // f(i, column of the slice) for ids that fall into it
    int c0 = 0, c1 = 0, b0 = 0, b1 = 0;
    if (PENAL) span_of(r.ctx_start, row, r.n_ctx, c0, c1);
    if (BIAS) span_of(r.bias_start, row, r.n_bias, b0, b1);
    auto scan = [&](const int *ids, int begin, int end, auto f) {
#pragma unroll 4
        for (int i = begin + t; i < end; i += kTableThreads) {
            const int id = ids[i];
            const unsigned at = (unsigned)(id - v0);
            if (id >= 0 && at < (unsigned)n) f(i, at);
        }
    };
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    long long made = 0;
    if (PENAL) {
        if (r.rep_penalty) rep = r.rep_penalty[row];
        if (r.frequency) freq = r.frequency[row];
        if (r.presence) pres = r.presence[row];
        made = (long long)c0 + (r.n_prompt ? max(r.n_prompt[row], 0) : 0);
        if (!(rep > 0.0f)) rep = 1.0f;
    }
    auto number_columns = [&] {
        for (int i = t; i < words; i += kTableThreads) map[i] = 0;
        table_sync();
        auto mark = [&](int, unsigned at) { atomicOr(&map[at >> 5], 1u << (at & 31)); };
        if (PENAL) scan(r.ctx, c0, c1, mark);
        if (BIAS) scan(r.bias_ids, b0, b1, mark);
        table_sync();
        const int per = (words + kTableThreads - 1) / kTableThreads, w0 = min(words, t * per), w1 = min(words, w0 + per);
        unsigned mine = 0;
        for (int w = w0; w < w1; ++w) mine += __popc(map[w]);
        unsigned sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned x = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += x;
        }
        if (lane == 31) warp_sum[t >> 5] = sum;
        table_sync();
        unsigned ahead = sum - mine, all = 0;
#pragma unroll
        for (int i = 0; i < kTableThreads / 32; ++i) {
            const unsigned x = warp_sum[i];
            if (i < (t >> 5)) ahead += x;
            all += x;
        }
        for (int w = w0; w < w1; ++w) {
            before[w] = ahead;
            ahead += __popc(map[w]);
        }
        if (t == 0) touched_s = all;
    };
    // counts and pairs of the touched columns numbered base .. base + kTouched - 1
    auto build = [&](unsigned base) {
        for (int i = t; i < kTouched; i += kTableThreads) {
            if (PENAL) count[i] = 0;
            if (BIAS) pair[i] = -1;
        }
        table_sync();
        auto number = [&](unsigned at) { return before[at >> 5] + __popc(map[at >> 5] & ((1u << (at & 31)) - 1)) - base; };
        if (PENAL)
            scan(r.ctx, c0, c1, [&](int i, unsigned at) {
                const unsigned k = number(at);
                if (k < kTouched) {
                    list[k] = (int)at;   // the same whoever writes it
                    atomicOr(&count[k], kSeen);
                    if (i >= made) atomicAdd(&count[k], 1u);
                }
            });
        if (BIAS)
            scan(r.bias_ids, b0, b1, [&](int i, unsigned at) {
                const unsigned k = number(at);
                if (k < kTouched) {
                    list[k] = (int)at;
                    atomicMax(&pair[k], i);
                }
            });
    };
    if (t == 0) next = 0;
    __syncthreads();
    if (SPARSE && t < kTableThreads) {
        number_columns();
        build(0);
    }

    // ---- the copy, a step of a warp at a time
    for (;;) {
        int step = 0;
        if (lane == 0) step = atomicAdd(&next, 1);
        step = __shfl_sync(0xffffffffu, step, 0);
        if (step * kStep >= n) break;
        const int first = v0 + step * kStep;
        auto column = [&](int i) { return first + i * 128 + lane * 4; };
        auto whole = [&](int c) { return c >= 0 && c + 3 < v0 + n; };
        float4 l[kVecs];
        unsigned words_of = 0;   // lane x: mask word first / 32 + x (0 outside the mask)
        if (MASK) {
            const int w = (first >> 5) + lane;
            if (lane <= kStep / 32 + 1 && w >= 0 && w <= (a.V - 1) >> 5) words_of = mask[w];
        }
        if (!in_place) {
#pragma unroll
            for (int i = 0; i < kVecs; ++i) {
                const int c = column(i);
                if (same && whole(c)) {
                    l[i] = __ldcs(reinterpret_cast<const float4 *>(in + c));
                } else {
                    float *e = &l[i].x;
#pragma unroll
                    for (int j = 0; j < 4; ++j) e[j] = c + j >= 0 && c + j < v0 + n ? in[c + j] : 0.0f;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            const int c = column(i);
            float *e = &l[i].x;
            unsigned ok = 15u;
            if (MASK) {   // bits c .. c + 3
                const int w = (c >> 5) - (first >> 5);
                const unsigned lo = __shfl_sync(0xffffffffu, words_of, w), hi = __shfl_sync(0xffffffffu, words_of, w + 1);
                ok = __funnelshift_r(lo, hi, c & 31) & 15u;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (!((ok >> j) & 1u)) e[j] = G2_MASKED;
            }
            if (in_place && ok == 15u) continue;
            if (whole(c) && (!in_place || ok == 0)) {
                __stcs(reinterpret_cast<float4 *>(out + c), l[i]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c + j >= 0 && c + j < v0 + n && (!in_place || !((ok >> j) & 1u))) out[c + j] = e[j];
            }
        }
    }
    if (!SPARSE) return;
    // ---- the touched columns, after their copies
    __syncthreads();
    const unsigned touched = touched_s;
    for (unsigned base = 0; base < touched; base += kTouched) {
        if (base > 0) {
            if (t < kTableThreads) build(base);
            __syncthreads();
        }
        for (unsigned k = t; k < min((unsigned)kTouched, touched - base); k += kRuleThreads) {
            const int c = v0 + list[k];
            if (MASK && !((mask[c >> 5] >> (c & 31)) & 1u)) continue;
            float x = in[c];
            if (PENAL && (count[k] & kSeen)) {
                x = x > 0.0f ? x / rep : x * rep;
                if (count[k] & kCount) {
                    x -= freq * (float)(count[k] & kCount);
                    x -= pres;
                }
            }
            if (BIAS && pair[k] >= 0) x += r.bias[pair[k]];
            out[c] = x;
        }
        __syncthreads();
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

cudaError_t launch_rules(const float *logits, long long ld, float *out, long long ld_out, int rows, int vocab,
                         const g2_logit_rules &rules, cudaStream_t st) {
    const int sms = sm_count();
    const int columns = vocab + 3;   // 3: a row that begins past a multiple of 16 bytes
    // equal slices, about eight for each SM over all rows, in waves of five (256 rows of 50257: four 27.7 us, one wave;
    // eight 25.6, two waves of which the second is 73% full; sixteen 30.6)
    const int fewest = (columns + kMaxSlice - 1) / kMaxSlice, most = (columns + kMinSlice - 1) / kMinSlice;
    const int slices = std::min(std::max((8 * sms + rows - 1) / rows, fewest), most);
    const int slice = ((columns + slices - 1) / slices + 127) / 128 * 128;
    const RuleArgs a{logits, out, ld, ld_out, vocab, slice, rules};
    const dim3 grid((columns + slice - 1) / slice, rows);
    const bool penal = rules.n_ctx > 0 && (rules.rep_penalty || rules.presence || rules.frequency), bias = rules.n_bias > 0;
    void (*const kernels[8])(RuleArgs) = {
        rules_kernel<false, false, false>, rules_kernel<true, false, false>, rules_kernel<false, true, false>, rules_kernel<true, true, false>,
        rules_kernel<false, false, true>,  rules_kernel<true, false, true>,  rules_kernel<false, true, true>,  rules_kernel<true, true, true>};
    return launch_pdl(kernels[(penal ? 1 : 0) + (bias ? 2 : 0) + (rules.mask ? 4 : 0)], grid, dim3(kRuleThreads), penal || bias ? slice / 4 : 0, st, a);
}

}  // namespace g2

using namespace g2;

extern "C" int g2k_process_logits(const float *logits, long long ld, float *out, long long ld_out, int rows, int vocab_size,
                                  const g2_logit_rules *rules, void *stream) {
    const char *who = "g2k_process_logits";
    if (!logits || !out) return arg_error(G2_ERR_ARG, who, "null argument");
    if (rows < 0 || rows > 65535 || vocab_size < 1 || vocab_size > 1 << 30)
        return arg_error(G2_ERR_RANGE, who, "need 0 <= rows <= 65535 and 1 <= vocab_size <= 2^30");
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
    return launch_status(who, launch_rules(logits, ld, out, ld_out, rows, vocab_size, *rules, (cudaStream_t)stream));
}
