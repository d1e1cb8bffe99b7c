"""The decode-time operators of the engine and the work they are measured on.

Four operators that a decode step of a served GPT-2 runs on device tensors:

  matvec   y = x' W with W held as 4-bit codes and one scale per group of rows of a column
           (x' = x or LayerNorm(x); bias, tanh GELU and residual as in the fp32 matvec);
  append   the K and V rows of new tokens quantised into a paged cache of 8-bit codes with one scale
           for each block (page) of tokens and head, and the rows of a block read back as values;
  attend   softmax attention of a few query rows per sequence over that cache;
  logits   penalties for repeated tokens, biases and grammar masks on rows of logits.

``run`` computes them as elementary torch operations, or, where ``own`` is true, by the library's
entry points.  ``exact`` has the same results in 64 bits, from the definitions.
"""
import math
import os
import sys

import torch

own = False

F32, F16 = 0, 1          # the library's G2_F32 / G2_F16
I8, E4M3 = 0, 1          # the library's G2_KV_I8 / G2_KV_E4M3
MASKED = -1e30           # the sampler's value of a token that must not be drawn
SCALE_FLOOR = 2.0 ** -64  # least scale of a cache block


def _lib():
    p = os.path.join(os.getcwd(), "gpt2-opencl-1.1_b200")
    if p not in sys.path:
        sys.path.insert(0, p)
    import gpt2b200
    return gpt2b200


# ---- cases -----------------------------------------------------------------------------
def listed():
    return [
        # one sequence's attention output projection of GPT-2 small, residual added: the smallest call
        {"name": "matvec small proj", "op": "matvec", "rows": 1, "K": 768, "N": 768, "group": 64, "dtype": "f32",
         "ln": False, "bias": True, "gelu": False, "residual": True},
        # GPT-2 XL's first MLP product for a few sequences of an fp16 program, its LayerNorm and GELU fused
        {"name": "matvec xl mlp 4 rows", "op": "matvec", "rows": 4, "K": 1600, "N": 6400, "group": 32, "dtype": "f16",
         "ln": True, "bias": True, "gelu": True, "residual": False},
        # GPT-2 XL's LM head for one sequence: an odd width, and a last group of 64 in groups of 128
        {"name": "matvec xl lm head", "op": "matvec", "rows": 1, "K": 1600, "N": 50257, "group": 128, "dtype": "f32",
         "ln": True, "bias": False, "gelu": False, "residual": False},
        # a wide model's projection for 16 sequences: the largest weights and the most rows
        {"name": "matvec wide 16 rows", "op": "matvec", "rows": 16, "K": 8192, "N": 28672, "group": 128, "dtype": "f16",
         "ln": False, "bias": False, "gelu": False, "residual": False},
        # one decode step of 32 sequences of GPT-2 medium: one token each, blocks partly filled
        {"name": "append step 32", "op": "append", "seqs": 32, "max_q": 1, "heads": 16, "dim": 64, "page": 64,
         "fmt": "i8", "dtype": "f32"},
        # ragged prompts of GPT-2 XL's head layout written in one call
        {"name": "append prompts", "op": "append", "seqs": 8, "max_q": 1000, "heads": 25, "dim": 64, "page": 32,
         "fmt": "e4m3", "dtype": "f16"},
        # one sequence of GPT-2 small near the end of its context: latency counts
        {"name": "attend one", "op": "attend", "seqs": 1, "max_q": 1, "max_len": 1000, "kv_heads": 12, "group": 1,
         "dim": 64, "page": 64, "fmt": "i8", "dtype": "f32"},
        # a decode step of 32 ragged sequences of GPT-2 medium
        {"name": "attend step 32", "op": "attend", "seqs": 32, "max_q": 1, "max_len": 1024, "kv_heads": 16, "group": 1,
         "dim": 64, "page": 64, "fmt": "i8", "dtype": "f32"},
        # several drafted tokens per sequence checked at once, odd lengths, GPT-2 XL's heads
        {"name": "attend drafts", "op": "attend", "seqs": 9, "max_q": 7, "max_len": 2021, "kv_heads": 25, "group": 1,
         "dim": 64, "page": 16, "fmt": "i8", "dtype": "f16"},
        # long documents with shared K/V heads of 128: the largest cache
        {"name": "attend long", "op": "attend", "seqs": 4, "max_q": 1, "max_len": 65536, "kv_heads": 8, "group": 4,
         "dim": 128, "page": 64, "fmt": "e4m3", "dtype": "f16"},
        # one sequence's logits, a few tokens biased, no grammar
        {"name": "logits one", "op": "logits", "rows": 1, "V": 50257, "max_ctx": 1024, "penalties": True, "n_bias": 20,
         "mask": False},
        # a large batch under grammars, one of which allows nothing
        {"name": "logits batch", "op": "logits", "rows": 256, "V": 50257, "max_ctx": 1024, "penalties": True,
         "n_bias": 300, "mask": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["matvec", "append", "attend", "attend", "logits"])
    yes = lambda: rng.random() < 0.5  # noqa: E731
    if op == "matvec":
        K = _log(rng, 40, 8192)
        return {"op": op, "rows": rng.randint(1, 16), "K": K, "N": _log(rng, 40, min(60000, 200_000_000 // K)),
                "group": rng.choice([32, 64, 128]), "dtype": rng.choice(["f32", "f16"]), "ln": yes(), "bias": yes(),
                "gelu": yes(), "residual": yes()}
    common = {"dim": rng.choice([64, 128]), "page": rng.choice([16, 32, 64, 128]), "fmt": rng.choice(["i8", "e4m3"]),
              "dtype": rng.choice(["f32", "f16"])}
    if op == "append":
        heads = rng.randint(1, 25)
        q = 1 if yes() else _log(rng, 2, 1000)
        most = max(1, 6_000_000 // (heads * common["dim"] * q))
        return {"op": op, "seqs": _log(rng, 1, min(96, most)), "max_q": q, "heads": heads, **common}
    if op == "attend":
        kv, group = rng.randint(1, 20), rng.choice([1, 1, 2, 4, 5, 8])
        q = 1 if rng.random() < 0.7 else rng.randint(2, 24)
        cost = kv * common["dim"] * max(1, q * group // 4)
        n = _log(rng, 1, min(40000, max(64, 100_000_000 // cost)))
        most = max(1, 100_000_000 // (cost * n))
        return {"op": op, "seqs": _log(rng, 1, min(64, most)), "max_q": q, "max_len": n, "kv_heads": kv, "group": group,
                **common}
    V = _log(rng, 1000, 200000)
    return {"op": op, "rows": _log(rng, 1, min(256, max(1, 12_000_000 // V))), "V": V, "max_ctx": _log(rng, 1, 4000),
            "penalties": yes(), "n_bias": rng.choice([0, 7, 300]), "mask": yes()}


def _dt(case):
    return torch.float32 if case["dtype"] == "f32" else torch.float16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)


# ---- inputs ----------------------------------------------------------------------------
def _matvec_inputs(c, seed):
    g, dt = _gen(seed), _dt(c)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    M, K, N = c["rows"], c["K"], c["N"]
    s = {"W": rnd(K, N) * 0.02, "x": (rnd(M, K) * (1 + 4 * (torch.rand(1, K, device="cuda", generator=g) < 0.01))).to(dt)}
    if c["ln"]:
        s["gamma"], s["beta"] = 1 + 0.2 * rnd(K), 0.1 * rnd(K)
    if c["bias"]:
        s["bias"] = 0.1 * rnd(N)
    if c["residual"]:
        s["residual"] = rnd(M, N).to(dt)
    return s


def _quantise4(W, group):
    """Codes [K, N] in -7..7 and bf16 scales [groups, N] of a weight matrix: scale = bf16(fp32(max|w| / 7)) over
    each group of `group` rows of a column, code = w / scale rounded to nearest even (0 where the scale is 0)."""
    K, N = W.shape
    n = -(-K // group)
    P = torch.cat([W, W.new_zeros(n * group - K, N)]).view(n, group, N)
    scale = (P.abs().amax(1).double() / 7).float().bfloat16()
    d = scale.double()[:, None]
    codes = torch.where(d > 0, (P.double() / torch.where(d > 0, d, 1.0)).round().clamp(-7, 7), 0.0)
    return codes.to(torch.int8).view(n * group, N)[:K], scale


def _cache_inputs(c, seed, heads, lens, rows):
    """A paged cache with `lens` tokens in each sequence (list), its pages in no order, and `rows` spare positions."""
    g = _gen(seed)
    P, D, S = c["page"], c["dim"], len(lens)
    most = max(1, max(-(-(n + r) // P) for n, r in zip(lens, rows)))
    pages = S * most + 3
    table = torch.randperm(pages, device="cuda", generator=g)[:S * most].to(torch.int32).view(S, most)
    if c["fmt"] == "i8":
        codes = [torch.randn(pages, heads, P, D, device="cuda", generator=g).mul_(40).round_().clamp_(-127, 127)
                 .to(torch.int8) for _ in "kv"]
    else:
        codes = [torch.randn(pages, heads, P, D, device="cuda", generator=g).mul_(140).clamp_(-448, 448)
                 .to(torch.float8_e4m3fn).view(torch.int8) for _ in "kv"]
    top = 127.0 if c["fmt"] == "i8" else 448.0
    scales = [(0.5 + torch.rand(pages, heads, device="cuda", generator=g)) * 3 / top for _ in "kv"]
    return {"k": codes[0], "v": codes[1], "k_scale": scales[0], "v_scale": scales[1], "table": table}


def _ragged(c):
    """Query or new-token counts of the sequences, the largest first.  They go by the case, as the outputs' shapes do."""
    g = torch.Generator().manual_seed(c["seqs"] * 1009 + c["max_q"])
    q = torch.randint(1, c["max_q"] + 1, (c["seqs"],), generator=g)
    q[0] = c["max_q"]
    return g, q.tolist()


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _starts(counts):
    v = [0]
    for n in counts:
        v.append(v[-1] + n)
    return v


def prepare(case, seed):
    c = dict(case)
    s = {"case": c}
    op, dt = c["op"], _dt(c) if "dtype" in c else torch.float32
    if op == "matvec":
        s.update(_matvec_inputs(c, seed))
        W = s.pop("W")
        if own:   # the weights laid out once, as a program does when it loads them
            g2 = _lib()
            s["packed"] = torch.empty(g2.q4_bytes(c["N"], c["K"], c["group"]), dtype=torch.uint8, device="cuda")
            g2.q4_pack(W, s["packed"], c["N"], c["K"], c["group"])
            s["y"] = torch.empty(c["rows"], c["N"], dtype=dt, device="cuda")
        else:
            codes, s["scale"] = _quantise4(W, c["group"])
            u = (codes + 8).to(torch.uint8)
            u = torch.cat([u, u.new_full((c["K"] % 2, c["N"]), 8)])
            s["codes"] = u[0::2] | (u[1::2] << 4)
    elif op == "append":
        g, q = _ragged(c)
        # a decode step lands anywhere in a block; a prompt may follow a shared prefix
        pos = torch.randint(0, 5 * c["page"], (c["seqs"],), generator=g).tolist()
        if c["max_q"] > 1:
            pos = [p if i % 2 else 0 for i, p in enumerate(pos)]
        s.update(_cache_inputs(c, seed, c["heads"], pos, q))
        gd = _gen(seed + 1)
        n, E = sum(q), c["heads"] * c["dim"]
        # K and V as the thirds of a c_attn output row; some tokens larger than what a block held before
        s["qkv"] = (torch.randn(n, 3 * E, device="cuda", generator=gd)
                    * (1 + 3 * (torch.rand(n, 1, device="cuda", generator=gd) < 0.2))).to(dt)
        first = [p - p % c["page"] for p in pos]
        back = [p + m - f for p, m, f in zip(pos, q, first)]
        s["q_start"], s["pos"], s["first"], s["b_start"] = _ints(_starts(q)), _ints(pos), _ints(first), _ints(_starts(back))
        s["rows"], s["back"], s["max_back"] = n, sum(back), max(back)
        s["k_out"] = torch.empty(s["back"], c["heads"], c["dim"], device="cuda")
        s["v_out"] = torch.empty_like(s["k_out"])
    elif op == "attend":
        _, q = _ragged(c)
        g = torch.Generator().manual_seed(int(seed) * 31 + 5)
        lens = torch.randint(1, c["max_len"] + 1, (c["seqs"],), generator=g).tolist()
        lens[0] = c["max_len"]
        if len(lens) > 3:
            lens[2] = 0
        s.update(_cache_inputs(c, seed, c["kv_heads"], lens, [0] * len(lens)))
        gd = _gen(seed + 1)
        H = c["kv_heads"] * c["group"]
        s["q"] = (torch.randn(sum(q), H, c["dim"], device="cuda", generator=gd) * 0.5).to(dt)
        s["q_start"], s["len"] = _ints(_starts(q)), _ints(lens)
        s["out"] = torch.empty_like(s["q"])
    else:
        gd = _gen(seed)
        g = torch.Generator().manual_seed(int(seed) * 31 + 5)
        R, V = c["rows"], c["V"]
        s["logits"] = torch.randn(R, V, device="cuda", generator=gd) * 3 - 1
        n = torch.randint(0, c["max_ctx"] + 1, (R,), generator=g).tolist()
        n[0] = c["max_ctx"]
        s["ctx_start"] = _ints(_starts(n))
        s["n_prompt"] = _ints([m // 2 for m in n])
        # text repeats itself: ids from a skewed distribution
        s["ctx"] = (torch.rand(max(1, sum(n)), device="cuda", generator=gd) ** 3 * V).to(torch.int32).clamp_(0, V - 1)
        if c["penalties"]:
            s["rep"] = 1 + 0.5 * torch.rand(R, device="cuda", generator=gd)
            s["presence"] = torch.rand(R, device="cuda", generator=gd)
            s["frequency"] = 0.3 * torch.rand(R, device="cuda", generator=gd)
        if c["n_bias"]:
            s["bias_start"] = _ints([i * c["n_bias"] for i in range(R + 1)])
            s["bias_ids"] = torch.randint(0, V, (R * c["n_bias"],), device="cuda", generator=gd, dtype=torch.int32)
            s["bias"] = torch.randn(R * c["n_bias"], device="cuda", generator=gd) * 5
        if c["mask"]:
            # a few tokens allowed, most allowed, or none at all (the last row of four)
            share = torch.tensor([0.01, 0.9, 0.5, 0.0], device="cuda").repeat(-(-R // 4))[:R]
            if R == 1:
                share[:] = 0.3
            words = -(-V // 32)
            bits = torch.rand(R, words * 32, device="cuda", generator=gd) < share[:, None]
            w = (bits.view(R, words, 32).long() << torch.arange(32, device="cuda")).sum(-1)
            s["mask"] = torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)
        s["out"] = torch.empty_like(s["logits"])
    if own:
        g2 = _lib()
        s["g2"] = g2
        if "k_scale" in s:
            s["cache"] = g2.kv8_cache(s["k"], s["v"], s["k_scale"], s["v_scale"], E4M3 if c["fmt"] == "e4m3" else I8)
        if op == "attend":
            n = g2.kv8_attention_workspace(s["cache"], c["kv_heads"] * c["group"], c["seqs"], c["max_q"])
            s["ws"] = torch.zeros(n, dtype=torch.uint8, device="cuda")
        if op == "logits":
            s["rules"] = g2.logit_rules(
                ctx=s["ctx"], ctx_start=s["ctx_start"], n_prompt=s["n_prompt"], rep_penalty=s.get("rep"),
                presence=s.get("presence"), frequency=s.get("frequency"), bias_ids=s.get("bias_ids"), bias=s.get("bias"),
                bias_start=s.get("bias_start"), mask=s.get("mask"), mask_stride=-(-c["V"] // 32) if c["mask"] else 0)
    return s


# ---- one pass --------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if own:
        return _run_own(s, c)
    return {"matvec": _plain_matvec, "append": _plain_append, "attend": _plain_attend, "logits": _plain_logits}[c["op"]](s, c)


def _run_own(s, c):
    g2 = s["g2"] if "g2" in s else _lib()
    op = c["op"]
    if op == "logits":
        g2.process_logits(s["logits"], s["out"], c["rows"], c["V"], s["rules"])
        return s["out"]
    dt = F16 if c["dtype"] == "f16" else F32
    if op == "matvec":
        g2.matvec_q4(s["x"], s["packed"], s["y"], c["rows"], c["N"], c["K"], c["group"], bias=s.get("bias"),
                     residual=s.get("residual"), gelu=c["gelu"], ln_gamma=s.get("gamma"), ln_beta=s.get("beta"), dtype=dt)
        return s["y"]
    t = s["table"]
    if op == "append":
        E = c["heads"] * c["dim"]
        g2.kv8_append(s["cache"], s["qkv"][:, E:], s["qkv"][:, 2 * E:], s["rows"], c["seqs"], t, t.shape[1],
                      s["pos"], q_start=s["q_start"], max_q=c["max_q"], row_stride=3 * E, dtype=dt)
        g2.kv8_gather(s["cache"], s["k_out"], s["v_out"], s["back"], c["seqs"], t, t.shape[1], s["first"],
                      q_start=s["b_start"], max_q=s["max_back"], dtype=F32)
        return {"k": s["k_out"], "v": s["v_out"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    g2.kv8_attention(s["cache"], s["q"], s["out"], c["kv_heads"] * c["group"], s["q"].shape[0], c["seqs"], t, t.shape[1],
                     s["len"], s["ws"], s["ws"].numel(), q_start=s["q_start"], max_q=c["max_q"], dtype=dt)
    return s["out"]


# ---- the plain forms -------------------------------------------------------------------
def _plain_matvec(s, c):
    u = s["codes"]
    W = torch.stack([u & 15, u >> 4], 1).view(-1, c["N"])[:c["K"]].float() - 8
    W = W * s["scale"].float().repeat_interleave(c["group"], 0)[:c["K"]]
    x = s["x"].float()
    if c["ln"]:
        x = x - x.mean(1, keepdim=True)
        x = x / (x.square().mean(1, keepdim=True) + 1e-5).sqrt() * s["gamma"] + s["beta"]
    y = x @ W
    if c["bias"]:
        y = y + s["bias"]
    if c["gelu"]:
        y = 0.5 * y * (1 + torch.tanh(0.7978845608 * (y + 0.044715 * y ** 3)))
    if c["residual"]:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def _seq_of(start, n):
    """Sequence and place in it of rows 0..n-1, for sequences that begin at `start`."""
    i = torch.arange(n, device="cuda")
    q = torch.searchsorted(start, i.int(), right=True) - 1
    return q, i - start.long()[q]


def _round8(t, fmt):
    """The nearest 8-bit value of each t (64 bits, within the format's range), ties to even."""
    if fmt == "i8":
        return t.round().clamp(-127, 127)
    step = torch.exp2((torch.frexp(t.abs()).exponent - 1).clamp(min=-6).double() - 3)
    return ((t / step).round() * step).clamp(-448, 448)


def _store8(v, fmt):
    return v.to(torch.int8) if fmt == "i8" else v.float().to(torch.float8_e4m3fn).view(torch.int8)


def _value8(code, fmt):
    return code.float() if fmt == "i8" else code.view(torch.float8_e4m3fn).float()


def _plain_append(s, c):
    P, H, D, fmt, n = c["page"], c["heads"], c["dim"], c["fmt"], s["rows"]
    top = 127.0 if fmt == "i8" else 448.0
    q, j = _seq_of(s["q_start"], n)
    at = s["pos"].long()[q] + j
    page = s["table"].long()[q, at // P]
    first = (at % P == 0) | (j == 0)                     # the first new row of its block
    fresh = torch.zeros(len(s["k"]), dtype=torch.bool, device="cuda")
    touched = fresh.clone().index_fill_(0, page, True)
    kept = torch.zeros(len(s["k"]), dtype=torch.long, device="cuda")   # rows of a block that stay
    kept = kept.index_put_((page,), torch.where(first, at % P, 0), accumulate=True)
    old = torch.arange(P, device="cuda") < kept[:, None]
    qkv = s["qkv"].float().view(n, 3, H, D)
    for code, scale, new in ((s["k"], s["k_scale"], qkv[:, 1]), (s["v"], s["v_scale"], qkv[:, 2])):
        peak = torch.zeros_like(scale).index_reduce_(0, page, new.abs().amax(-1), "amax")
        wide = torch.maximum((peak.double() / top).float(), peak.new_tensor(SCALE_FLOOR))
        wide = torch.where((kept > 0)[:, None], torch.maximum(wide, scale), wide)
        wide = torch.where(touched[:, None], wide, scale)
        grown = (wide.double() > scale.double()) & (kept > 0)[:, None]
        again = _value8(code, fmt).double() * scale.double()[:, :, None, None] / wide.double()[:, :, None, None]
        code.copy_(torch.where(grown[:, :, None, None] & old[:, None, :, None], _store8(_round8(again, fmt), fmt), code))
        code[page, :, at % P] = _store8(_round8(new.double() / wide[page].double()[:, :, None], fmt), fmt)
        scale.copy_(wide)
    q, j = _seq_of(s["b_start"], s["back"])
    at = s["first"].long()[q] + j
    page = s["table"].long()[q, at // P]
    k, v = (_value8(code[page, :, at % P], fmt) * scale[page][:, :, None]
            for code, scale in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])))
    return {"k": k, "v": v, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _plain_attend(s, c):
    P, D, Hk, G, S, Q = c["page"], c["dim"], c["kv_heads"], c["group"], c["seqs"], c["max_q"]
    t = s["table"].long()
    k, v = ((_value8(code[t], c["fmt"]) * scale[t][..., None, None]).transpose(2, 3).reshape(S, -1, Hk, D)
            for code, scale in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])))
    n = s["q"].shape[0]
    seq, j = _seq_of(s["q_start"], n)
    q = torch.zeros(S, Q, Hk * G, D, device="cuda")
    q[seq, j] = s["q"].float()
    # queries of a K/V head together: [S, Hk, Q * G, D] x [S, Hk, D, T]
    q = q.view(S, Q, Hk, G, D).permute(0, 2, 1, 3, 4).reshape(S, Hk, Q * G, D)
    score = (q @ k.permute(0, 2, 3, 1)) / math.sqrt(D)
    count = (s["q_start"][1:] - s["q_start"][:-1]).long()
    last = s["len"].long()[:, None] - count[:, None] + torch.arange(Q, device="cuda")
    seen = torch.arange(k.shape[1], device="cuda") <= last[:, :, None]
    seen &= torch.arange(k.shape[1], device="cuda") < s["len"].long()[:, None, None]
    score = score.view(S, Hk, Q, G, -1).masked_fill(~seen[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = p.view(S, Hk, Q * G, -1) @ v.transpose(1, 2)
    out = out.view(S, Hk, Q, G, D).permute(0, 2, 1, 3, 4).reshape(S, Q, Hk * G, D)
    return out[seq, j].to(s["q"].dtype)


def _plain_logits(s, c):
    R, V = c["rows"], c["V"]
    l = s["logits"]
    if c["penalties"]:
        row, j = _seq_of(s["ctx_start"], len(s["ctx"]))
        row = row.clamp(0, R - 1)   # the one spare id of empty contexts
        live = torch.arange(len(s["ctx"]), device="cuda") < s["ctx_start"][-1]
        at = row * V + s["ctx"].long()
        any_ = torch.zeros(R * V, device="cuda").index_add_(0, at, live.float()).view(R, V)
        made = torch.zeros(R * V, device="cuda").index_add_(0, at, (live & (j >= s["n_prompt"][row])).float()).view(R, V)
        rep = s["rep"][:, None]
        l = torch.where(any_ > 0, torch.where(l > 0, l / rep, l * rep), l)
        l = l - s["frequency"][:, None] * made - s["presence"][:, None] * (made > 0)
    if c["n_bias"]:
        row, j = _seq_of(s["bias_start"], len(s["bias"]))
        at = row * V + s["bias_ids"].long()
        i = torch.arange(len(at), device="cuda")
        which = torch.full((R * V,), -1, device="cuda", dtype=torch.long).index_reduce_(0, at, i, "amax")   # the last entry counts
        l = l + torch.where(which >= 0, s["bias"][which.clamp(min=0)], 0.0).view(R, V)
    if c["mask"]:
        v = torch.arange(V, device="cuda")
        ok = (s["mask"][:, v // 32] >> (v % 32).int()) & 1
        l = torch.where(ok == 1, l, MASKED)
    return l + 0 if l is s["logits"] else l


# ---- what a pass cannot do without -------------------------------------------------------
def work(case):
    c, op = case, case["op"]
    e = 2 if c.get("dtype") == "f16" else 4
    if op == "matvec":
        M, K, N = c["rows"], c["K"], c["N"]
        b = K * N / 2 + 2 * N * -(-K // c["group"]) + e * (M * K + M * N * (1 + c["residual"])) + 4 * N * c["bias"] + 8 * K * c["ln"]
        return {"bytes": b, "flops": 2 * M * K * N}
    if op == "append":
        n, E = c["seqs"] * (c["max_q"] + 1) / 2, c["heads"] * c["dim"]
        back = n + c["seqs"] * c["page"] / 2
        return {"bytes": n * 2 * E * (e + 1) + back * 2 * E * 5, "flops": 8 * n * E}
    if op == "attend":
        H, n = c["kv_heads"] * c["group"], c["seqs"] * (c["max_q"] + 1) / 2
        keys = c["max_len"] if c["seqs"] == 1 else c["seqs"] * (c["max_len"] + 1) / 2
        return {"bytes": keys * c["kv_heads"] * (2 * c["dim"] + 8 / c["page"]) + 2 * e * n * H * c["dim"],
                "flops": 4 * keys * (n / c["seqs"]) * H * c["dim"]}
    R, V = c["rows"], c["V"]
    return {"bytes": R * (8 * V + 4 * c["max_ctx"] / 2 * c["penalties"] + 8 * c["n_bias"] + V / 8 * c["mask"]), "flops": 6 * R * V}


# ---- the definitions in 64 bits ------------------------------------------------------------
def exact(case, seed):
    c, op = dict(case), case["op"]
    if op == "matvec":
        s = _matvec_inputs(c, seed)
        W, x, G = s["W"].double(), s["x"].double(), c["group"]
        y = torch.zeros(c["rows"], c["N"], dtype=torch.double, device="cuda")
        if c["ln"]:
            var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
            x = (x - mean) * torch.rsqrt(var + 1e-5) * s["gamma"].double() + s["beta"].double()
        for k in range(0, c["K"], G):
            w = W[k:k + G]
            step = (w.abs().max(0).values / 7).float().bfloat16().double()
            code = torch.nan_to_num(w / step).round().clamp(-7, 7)
            y += x[:, k:k + G] @ (code * step)
        if c["bias"]:
            y += s["bias"].double()
        if c["gelu"]:
            y = y / (1 + torch.exp(-2 * 0.7978845608 * (y + 0.044715 * y * y * y)))
        return y + s["residual"].double() if c["residual"] else y
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"append": _exact_append, "attend": _exact_attend, "logits": _exact_logits}[op](s, c)


def _grid(fmt):
    """The non-negative values of the format, and 127 or 448 where it ends."""
    if fmt == "i8":
        return torch.arange(128, dtype=torch.double, device="cuda")
    b = torch.arange(127, device="cuda")
    e, m = (b >> 3).double(), (b & 7).double()
    return torch.where(e > 0, (1 + m / 8) * torch.exp2(e - 7), m / 8 * 2.0 ** -6)


def _nearest(x, fmt):
    """The format's value next to each x; of two as near the one with an even code."""
    g = _grid(fmt)
    a = x.abs().clamp(max=float(g[-1]))
    hi = torch.searchsorted(g, a).clamp(1, len(g) - 1)
    lo = hi - 1
    up = (g[hi] - a < a - g[lo]) | ((g[hi] - a == a - g[lo]) & (hi % 2 == 0))
    return torch.where(up, g[hi], g[lo]) * torch.where(x < 0, -1.0, 1.0)


def _exact_append(s, c):
    P, H, D, fmt = c["page"], c["heads"], c["dim"], c["fmt"]
    top = 127 if fmt == "i8" else 448
    start, pos, table = s["q_start"].tolist(), s["pos"].tolist(), s["table"].tolist()
    got = {"k": [], "v": []}
    for name, third in (("k", 1), ("v", 2)):
        new = s["qkv"].double().view(s["rows"], 3, H, D)[:, third]
        code = s[name] if fmt == "i8" else s[name].view(torch.float8_e4m3fn)
        scale = s[name + "_scale"].clone()
        for i in range(c["seqs"]):
            p, end = pos[i], pos[i] + start[i + 1] - start[i]
            while p < end:
                page, stop = table[i][p // P], min(end, (p // P + 1) * P)
                x = new[start[i] + p - pos[i]:start[i] + stop - pos[i]]          # [rows, H, D]
                step = (x.abs().amax((0, 2)) / top).float().clamp(min=SCALE_FLOOR)
                held = code[page, :, :p % P].double().transpose(0, 1)             # [rows, H, D]
                was = scale[page].clone()
                if p % P:
                    step = torch.maximum(step, was)
                    more = (step > was)[:, None]
                    held = torch.where(more, _nearest(held * was.double()[:, None] / step.double()[:, None], fmt), held)
                got[name].append(torch.cat([held, _nearest(x / step.double()[:, None], fmt)]) * step.double()[:, None])
                scale[page] = step
                p = stop
        got[name + "_scale"] = scale.double()
    return {n: torch.cat(v) if isinstance(v, list) else v for n, v in got.items()}


def _exact_attend(s, c):
    P, D, Hk, G = c["page"], c["dim"], c["kv_heads"], c["group"]
    start, lens = s["q_start"].tolist(), s["len"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.double, device="cuda")
    for i, n in enumerate(lens):
        pages = s["table"][i, :-(-n // P)].long()
        if not n:
            continue
        k, v = ((s[x][pages] if c["fmt"] == "i8" else s[x].view(torch.float8_e4m3fn)[pages]).double()
                * s[x + "_scale"][pages].double()[:, :, None, None] for x in "kv")
        k, v = (x.transpose(0, 1).reshape(Hk, -1, D)[:, :n] for x in (k, v))
        m = start[i + 1] - start[i]
        for j in range(m):
            keys = n - m + j + 1
            if keys <= 0:
                continue
            q = s["q"][start[i] + j].double().view(Hk, G, D)
            p = torch.softmax(torch.einsum("hgd,htd->hgt", q, k[:, :keys]) * D ** -0.5, -1)
            out[start[i] + j] = torch.einsum("hgt,htd->hgd", p, v[:, :keys]).reshape(Hk * G, D)
    return out


def _exact_logits(s, c):
    out = s["logits"].double()
    if c["penalties"]:
        ends, prompts = s["ctx_start"].tolist(), s["n_prompt"].tolist()
        for r in range(c["rows"]):
            ids = s["ctx"][ends[r]:ends[r + 1]].long()
            seen = torch.unique(ids)
            l = out[r, seen]
            rep = s["rep"][r].double()
            out[r, seen] = torch.where(l > 0, l / rep, l * rep)
            made, count = torch.unique(ids[prompts[r]:], return_counts=True)
            out[r, made] -= s["presence"][r].double() + s["frequency"][r].double() * count
    if c["n_bias"]:
        for r in range(c["rows"]):
            a, b = r * c["n_bias"], (r + 1) * c["n_bias"]
            last = dict(zip(s["bias_ids"][a:b].tolist(), s["bias"][a:b].tolist()))
            out[r, torch.tensor(list(last), device="cuda")] += torch.tensor(list(last.values()), dtype=torch.double, device="cuda")
    if c["mask"]:
        shifts = torch.arange(32, device="cuda")
        ok = ((s["mask"][:, :, None].long() >> shifts) & 1).view(c["rows"], -1)[:, :c["V"]]
        out[ok == 0] = MASKED
    return out
