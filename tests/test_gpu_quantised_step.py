"""The 4-bit matvec, the 8-bit paged cache, the logit rules and the top-k together:
decode steps of a small two-layer GPT-2 whose weights and cache are quantised.

Every operator's output is compared with its definition in 64 bits on the inputs
it really had (so that a code of the cache that falls on the other side of a
border does not count): a product of K terms to (K / 16 + 16) 2^-22 of sum |x| |w|
as in the operators' own tests, here with the 2-norms of rows (LayerNorm's sum is
bounded by its row's); attention to 2^-17 of the largest value, A <= 1 being below
the scores of this model.  Then the same steps run as a captured graph, in place
of eager calls, and must give the same tokens and the same bits.
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

S, E, H, L, V, P, BLOCKS, GROUP = 3, 128, 2, 2, 1009, 16, 6, 32
D = E // H


@pytest.fixture(scope="module")
def g2():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import gpt2b200
    return gpt2b200


class Weight:
    def __init__(self, g2, K, N, g):
        W = torch.randn(K, N, device="cuda", generator=g) * 0.05
        self.K, self.N = K, N
        self.packed = torch.empty(g2.q4_bytes(N, K, GROUP), dtype=torch.uint8, device="cuda")
        g2.q4_pack(W, self.packed, N, K, GROUP)
        values = torch.empty(K, N, device="cuda")
        g2.q4_unpack(self.packed, values, N, K, GROUP)
        self.values = values.double()
        self.bias = torch.randn(N, device="cuda", generator=g) * 0.1


def norm(x, ga, be):
    x = x.double()
    return (x - x.mean(-1, keepdim=True)) * (x.var(-1, correction=0, keepdim=True) + 1e-5).rsqrt() * ga.double() + be.double()


def gelu(y):
    return 0.5 * y * (1 + torch.tanh(0.7978845608 * (y + 0.044715 * y ** 3)))


class Model:
    def __init__(self, g2, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        self.g2 = g2
        self.wte, self.wpe = rnd(V, E) * 0.5, rnd(P * BLOCKS, E) * 0.1
        self.layers = [dict(qkv=Weight(g2, E, 3 * E, g), proj=Weight(g2, E, E, g), fc=Weight(g2, E, 4 * E, g),
                            fc2=Weight(g2, 4 * E, E, g), g1=1 + 0.1 * rnd(E), b1=0.1 * rnd(E), g2=1 + 0.1 * rnd(E), b2=0.1 * rnd(E))
                       for _ in range(L)]
        self.head, self.gf, self.bf = Weight(g2, E, V, g), 1 + 0.1 * rnd(E), 0.1 * rnd(E)
        pages = S * BLOCKS + 1
        self.caches = []
        for fmt in (g2.G2_KV_I8, g2.G2_KV_E4M3):     # a layer of each
            k, v = (torch.full((pages, H, P, D), 0x7f, dtype=torch.int8, device="cuda") for _ in "kv")
            ks, vs = (torch.full((pages, H), math.nan, device="cuda") for _ in "kv")
            self.caches.append(g2.kv8_cache(k, v, ks, vs, fmt))
        self.table = torch.randperm(pages, device="cuda", generator=g)[:S * BLOCKS].to(torch.int32).view(S, BLOCKS)
        self.ws = torch.zeros(g2.kv8_attention_workspace(self.caches[0], H, S, 1), dtype=torch.uint8, device="cuda")
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        new = lambda *s: torch.empty(*s, device="cuda")  # noqa: E731
        self.x, self.qkv, self.att, self.ffn, self.logits, self.ruled = new(S, E), new(S, 3 * E), new(S, E), new(S, 4 * E), new(S, V), new(S, V)
        self.top = new(S, 4)
        self.ids = torch.empty(S, 4, dtype=torch.int32, device="cuda")
        self.pos, self.len = (torch.zeros(S, dtype=torch.int32, device="cuda") for _ in "ab")
        # rules: penalties over the tokens made so far, a bias, a grammar without the even ids
        self.made = torch.zeros(S, 32, dtype=torch.int32, device="cuda")
        bits = (torch.arange(-(-V // 32) * 32, device="cuda") % 2 == 1).view(-1, 32).long()
        w = (bits << torch.arange(32, device="cuda")).sum(-1)
        self.mask = torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)
        self.start = torch.arange(S + 1, device="cuda", dtype=torch.int32) * 32
        three = lambda v: torch.full((S,), v, device="cuda")  # noqa: E731
        self.rules = g2.logit_rules(ctx=self.made, ctx_start=self.start, rep_penalty=three(1.3), presence=three(0.2), frequency=three(0.1),
                                    bias_ids=torch.tensor([7, 8, 9], device="cuda", dtype=torch.int32),
                                    bias=torch.tensor([2.0, 50.0, -1.0], device="cuda"),
                                    bias_start=torch.arange(S + 1, device="cuda", dtype=torch.int32), mask=self.mask)

    def step(self, check=None, stream=0):
        """One token of each sequence: embeds self.token at self.pos (length self.len after it)."""
        g2, c = self.g2, dict(stream=stream)
        see = check or (lambda *a: None)
        for w, cache in zip(self.layers, self.caches):
            g2.matvec_q4(self.x, w["qkv"].packed, self.qkv, S, 3 * E, E, GROUP, bias=w["qkv"].bias, ln_gamma=w["g1"], ln_beta=w["b1"], **c)
            see("qkv", norm(self.x, w["g1"], w["b1"]), w["qkv"], self.qkv)
            g2.kv8_append(cache, self.qkv[:, E:], self.qkv[:, 2 * E:], S, S, self.table, BLOCKS, self.pos, row_stride=3 * E, status=self.status, **c)
            g2.kv8_attention(cache, self.qkv, self.att, H, S, S, self.table, BLOCKS, self.len, self.ws, self.ws.numel(), q_stride=3 * E,
                             status=self.status, **c)
            see("attention", cache)
            before = self.x.clone() if check else None
            g2.matvec_q4(self.att, w["proj"].packed, self.x, S, E, E, GROUP, bias=w["proj"].bias, residual=self.x, **c)
            see("proj", self.att.double(), w["proj"], self.x, before)
            g2.matvec_q4(self.x, w["fc"].packed, self.ffn, S, 4 * E, E, GROUP, bias=w["fc"].bias, gelu=True, ln_gamma=w["g2"], ln_beta=w["b2"], **c)
            see("fc", norm(self.x, w["g2"], w["b2"]), w["fc"], self.ffn)
            before = self.x.clone() if check else None
            g2.matvec_q4(self.ffn, w["fc2"].packed, self.x, S, E, 4 * E, GROUP, bias=w["fc2"].bias, residual=self.x, **c)
            see("fc2", self.ffn.double(), w["fc2"], self.x, before)
        g2.matvec_q4(self.x, self.head.packed, self.logits, S, V, E, GROUP, ln_gamma=self.gf, ln_beta=self.bf, **c)
        g2.process_logits(self.logits, self.ruled, S, V, self.rules, **c)
        for s in range(S):
            g2.topk(self.ruled[s], V, 4, self.top[s], self.ids[s], **c)

    def embed(self, tokens):
        return self.wte[tokens.long()] + self.wpe[self.pos.long()]


def comparer(m):
    def see(name, *a):
        torch.cuda.synchronize()
        assert int(m.status) == 0
        if name == "attention":
            cache, n = a[0], int(m.len.max())
            pad = torch.zeros(S * n, H, D, device="cuda")
            k, v = pad.clone(), pad.clone()
            starts = torch.cat([torch.zeros(1, device="cuda", dtype=torch.int32), m.len.cumsum(0).int()])
            m.g2.kv8_gather(cache, k, v, S * n, S, m.table, BLOCKS, torch.zeros_like(m.pos), q_start=starts, max_q=n, status=m.status)
            for s in range(S):
                i, j = int(starts[s]), int(starts[s + 1])
                q = m.qkv[s, :E].double().view(H, D)
                p = (torch.einsum("hd,khd->hk", q, k[i:j].double()) * D ** -0.5).softmax(-1)
                want = torch.einsum("hk,khd->hd", p, v[i:j].double()).flatten()
                assert (m.att[s] - want).abs().max() <= 2 ** -17 * v[i:j].abs().max()
                # the newest rows are the thirds of c_attn's, to the cache's precision
                top = 127 if cache.format == m.g2.G2_KV_I8 else 16
                for out, part in ((k, 1), (v, 2)):
                    row = m.qkv[s, part * E:(part + 1) * E].view(H, D)
                    assert ((out[j - 1] - row).abs() <= out[i:j].abs().amax((0, 2))[:, None] / top).all()
            return
        x, w, y = a[0], a[1], a[2]
        want = x @ w.values + w.bias.double()
        size = x.norm(dim=-1, keepdim=True) * w.values.norm(dim=0) + w.bias.abs()
        if name == "fc":
            want, size = gelu(want), size * 1.2
        if len(a) > 3:
            want, size = want + a[3].double(), size + a[3].abs()
        assert ((y - want).abs() <= (w.K / 16 + 16) * 2 ** -22 * size).all(), name
    return see


def run(m, steps, graph=False, check=False):
    g = torch.Generator(device="cuda").manual_seed(5)
    m.pos.copy_(torch.tensor([0, 0, 0]))
    m.len.fill_(1)
    m.made.zero_()
    token = torch.tensor([11, 300, 777], device="cuda")
    see = comparer(m) if check else None
    exec_ = None
    if graph:
        exec_ = torch.cuda.CUDAGraph()
        with torch.cuda.graph(exec_):
            m.step(stream=torch.cuda.current_stream().cuda_stream)
    out = []
    for i in range(steps):
        m.x.copy_(m.embed(token))
        exec_.replay() if graph else m.step(see)
        torch.cuda.synchronize()
        token = m.ids[:, 0]
        assert (token % 2 == 1).all() and (m.ids == m.ruled.topk(4).indices).all()
        assert (m.ruled[:, 0::2] == -1e30).all() and (m.ruled[:, 1::2] > -1e29).all()
        out.append((m.ids.clone(), m.logits.clone(), m.ruled.clone()))
        m.made[:, i % 32] = token
        m.pos.add_(1)
        m.len.add_(1)
    assert int(m.status) == 0 and g is not None
    return out


def test_steps_against_the_definitions(g2):
    run(Model(g2), 35, check=True)


def test_captured_steps_are_the_eager_ones(g2):
    a, b = run(Model(g2), 60), run(Model(g2), 60, graph=True)
    for x, y in zip(a, b):
        assert all(torch.equal(p, q) for p, q in zip(x, y))


def test_prompt_then_steps(g2):
    """A prompt's rows written in one call hold the same values as written row by row into fresh blocks with the largest row first,
    and several rows of queries attend causally over them."""
    m = Model(g2, seed=1)
    cache, n = m.caches[0], 37
    g = torch.Generator(device="cuda").manual_seed(3)
    rows = torch.randn(n, 3 * E, device="cuda", generator=g)
    rows[0::P] *= 4                                                # the first row of a block has its largest value
    starts = torch.tensor([0, n], device="cuda", dtype=torch.int32)
    zero = torch.zeros(1, device="cuda", dtype=torch.int32)
    got = []
    for one_by_one in (False, True):
        if one_by_one:
            for i in range(n):
                g2.kv8_append(cache, rows[i:, E:], rows[i:, 2 * E:], 1, 1, m.table, BLOCKS, zero + i, row_stride=3 * E, status=m.status)
        else:
            g2.kv8_append(cache, rows[:, E:], rows[:, 2 * E:], n, 1, m.table, BLOCKS, zero, q_start=starts, max_q=n, row_stride=3 * E, status=m.status)
        k, v = torch.empty(n, E, device="cuda"), torch.empty(n, E, device="cuda")
        g2.kv8_gather(cache, k, v, n, 1, m.table, BLOCKS, zero, q_start=starts, max_q=n, status=m.status)
        got.append((k, v))
    assert int(m.status) == 0
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    out = torch.empty(n, E, device="cuda")
    ws = torch.zeros(g2.kv8_attention_workspace(cache, H, 1, n), dtype=torch.uint8, device="cuda")
    g2.kv8_attention(cache, rows, out, H, n, 1, m.table, BLOCKS, zero + n, ws, ws.numel(), q_start=starts, max_q=n, q_stride=3 * E)
    k, v = (x.view(n, H, D).double() for x in got[0])
    s = torch.einsum("qhd,khd->hqk", rows[:, :E].view(n, H, D).double(), k) * D ** -0.5
    p = s.masked_fill(torch.ones(n, n, device="cuda").triu(1).bool(), -math.inf).softmax(-1)
    want = torch.einsum("hqk,khd->qhd", p, v).reshape(n, E)
    assert (out - want).norm() <= 2 ** -15 * want.norm()
