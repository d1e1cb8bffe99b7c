"""The 8-bit paged KV cache on the GPU: g2k_kv8_append, g2k_kv8_gather and
g2k_kv8_attention against their definitions in 64 bits.

Writing is exact: scales and codes must equal, bit for bit, scale =
max(fp32(max|x| / 127 or 448), 2^-64) (at least the old one where rows stay) and
the nearest code of the exact quotient, ties to even.

Attention, with A the largest sum_d |q_d k_d| * scale of a row: a score is off
by at most (D / 16 + 8) 2^-22 A <= 2^-18 A (accumulation steps of a 64-bit-exact
product in fp32, the operands' split, the factor), a weight by that and 2^-21,
and the sum over n keys by (n / 16 + 16) 2^-22 of sum_j p_j |v_j|; so an output
by e = (2^-17 A + 2^-21 + (n / 16 + 16) 2^-22) * sum_j p_j |v_j|, plus half a step of its type.
A weight far below the largest is not carried to its own relative precision: fp32 has
none below 2^-126, and two fp16 parts end 2^-36 below the largest contribution p_j s_j
(s_j the page's V scale), 2^-24 for the first and 2^-12 of that for the second; each of n
weights times a code of at most 127 or 448 adds n 2^-35 max_j (p_j s_j) * 127 (or 448).
The 2-norm over all outputs is held to (1 + A) 2^-19 of the result's norm.
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

FMTS = ["i8", "e4m3"]
TOP = {"i8": 127.0, "e4m3": 448.0}
FLOOR = 2.0 ** -64


@pytest.fixture(scope="module")
def g2():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import gpt2b200
    return gpt2b200


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def grid(fmt):
    if fmt == "i8":
        return torch.arange(128, dtype=torch.double, device="cuda")
    b = torch.arange(127, device="cuda", dtype=torch.double)
    e, m = (b / 8).floor(), b % 8
    return torch.where(e > 0, (1 + m / 8) * torch.exp2(e - 7), m / 512)


def nearest(x, fmt):
    """Index-exact rounding to the format, through its table of values."""
    g = grid(fmt)
    a = x.abs().clamp(max=float(g[-1]))
    hi = torch.searchsorted(g, a).clamp(1, len(g) - 1)
    lo = hi - 1
    up = (g[hi] - a < a - g[lo]) | ((g[hi] - a == a - g[lo]) & (hi % 2 == 0))
    v = torch.where(up, g[hi], g[lo])
    return torch.where(x < 0, -v, v)


def values(code, fmt):
    return code.double() if fmt == "i8" else code.view(torch.float8_e4m3fn).double()


class Cache:
    """A cache of random codes, every page in use by nobody; scales and codes of free pages are hostile."""

    def __init__(self, g2, pages, heads, P, D, fmt, seed=0):
        g = gen(seed)
        self.g2, self.fmt, self.P, self.D, self.H = g2, fmt, P, D, heads
        self.k, self.v = (torch.randint(-128, 128, (pages, heads, P, D), device="cuda", generator=g).to(torch.int8) for _ in "kv")
        if fmt == "e4m3":
            self.k[..., ::7], self.v[..., ::5] = 0x7f, -1          # NaN codes
        self.ks, self.vs = (torch.full((pages, heads), math.nan, device="cuda") for _ in "kv")
        self.h = g2.kv8_cache(self.k, self.v, self.ks, self.vs, g2.G2_KV_E4M3 if fmt == "e4m3" else g2.G2_KV_I8)

    def fill(self, table, lens, seed=1, spread=1.0):
        """Finite codes and scales for the first lens[s] positions of each sequence; the rest stays hostile."""
        g = gen(seed)
        for s, n in enumerate(lens):
            for b in range(-(-n // self.P)):
                p, m = int(table[s, b]), min(self.P, n - b * self.P)
                for code, scale in ((self.k, self.ks), (self.v, self.vs)):
                    x = torch.randn(self.H, m, self.D, device="cuda", generator=g)
                    if self.fmt == "i8":
                        code[p, :, :m] = (x * 45).round().clamp(-127, 127).to(torch.int8)
                    else:
                        code[p, :, :m] = (x * 150).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.int8)
                    z = torch.randn(self.H, device="cuda", generator=g)
                    scale[p] = torch.exp2(z * spread) * 2 / TOP[self.fmt]


def tables(seqs, blocks, spare=2, seed=0):
    n = seqs * blocks + spare
    return n, torch.randperm(n, device="cuda", generator=gen(seed))[:seqs * blocks].to(torch.int32).view(seqs, blocks)


# ---- append ------------------------------------------------------------------------------
def model_append(cache, k, v, counts, pos, table):
    """Codes' values and scales after the call, from the definition; plain loops over blocks."""
    P, fmt = cache.P, cache.fmt
    out = []
    for code, scale, new in ((cache.k, cache.ks, k), (cache.v, cache.vs, v)):
        val, scale = values(code, fmt), scale.clone()
        row = 0
        for s, n in enumerate(counts):
            x_all = new[row:row + n].double()
            row += n
            p, end = pos[s], pos[s] + n
            while p < end:
                stop, page = min(end, (p // P + 1) * P), int(table[s, p // P])
                x, kept = x_all[p - pos[s]:stop - pos[s]].transpose(0, 1), p % P
                peak = x.abs().amax((1, 2))
                st = (peak / TOP[fmt]).float().clamp(min=FLOOR)
                st = torch.where(peak.isfinite(), st, math.nan)
                if kept:
                    was = scale[page].clone()
                    grown = st > was
                    st = torch.where(was.isnan(), was, torch.where(st < was, was, st))
                    old = val[page, :, :kept]
                    again = nearest(old * was.double()[:, None, None] / st.double()[:, None, None], fmt)
                    val[page, :, :kept] = torch.where(grown[:, None, None], again, old)
                q = nearest(x / st.double()[:, None, None], fmt)
                val[page, :, kept:kept + stop - p] = torch.where(st.isnan()[:, None, None], 0.0, q)
                scale[page] = st
                p = stop
        out.append((val, scale))
    return out


def same(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


def check_append(g2, cache, counts, pos, table, dtype="f32", seed=3, k=None, v=None, ragged=True, gather=True, stream=None):
    H, D, n = cache.H, cache.D, sum(counts)
    dt, code = (torch.float32, g2.G2_F32) if dtype == "f32" else (torch.float16, g2.G2_F16)
    g = gen(seed)
    E = H * D
    qkv = (torch.randn(n + 2, 3 * E, device="cuda", generator=g) * torch.exp2(torch.randn(n + 2, 1, device="cuda", generator=g))).to(dt)
    if k is not None:
        qkv[:n, E:2 * E], qkv[:n, 2 * E:] = k.reshape(n, E).to(dt), v.reshape(n, E).to(dt)
    kd, vd = qkv[:n, E:2 * E].reshape(n, H, D), qkv[:n, 2 * E:].reshape(n, H, D)
    want = model_append(cache, kd, vd, counts, pos, table)
    starts = [0]
    for c in counts:
        starts.append(starts[-1] + c)
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    kw = dict(q_start=ints(starts), max_q=max(max(counts), 1)) if ragged else {}
    g2.kv8_append(cache.h, qkv[:, E:], qkv[:, 2 * E:], n, len(counts), table, table.shape[1], ints(pos), row_stride=3 * E,
                  dtype=code, status=st, stream=0 if stream is None else stream, **kw)
    torch.cuda.synchronize()
    assert int(st) == 0
    for (val, scale), c, s in zip(want, (cache.k, cache.v), (cache.ks, cache.vs)):
        assert same(s, scale)
        assert same(values(c, cache.fmt), val)
    if gather:
        for od, oc in ((torch.float32, g2.G2_F32), (torch.float16, g2.G2_F16)):
            ko, vo = (torch.full((n + 1, H, D), 5.5, device="cuda", dtype=od) for _ in "kv")
            g2.kv8_gather(cache.h, ko, vo, n, len(counts), table, table.shape[1], ints(pos), dtype=oc, status=st, **kw)
            torch.cuda.synchronize()
            assert int(st) == 0 and (ko[n:] == 5.5).all() and (vo[n:] == 5.5).all()
            row = 0
            for s, c in enumerate(counts):
                for j in range(c):
                    p = pos[s] + j
                    page, t = int(table[s, p // cache.P]), p % cache.P
                    for o, (val, scale) in zip((ko, vo), want):
                        w = (val[page, :, t] * scale[page].double()[:, None]).to(od)
                        if od == torch.float16:
                            w = (val[page, :, t] * scale[page].double()[:, None]).float().to(od)
                        assert same(o[row + j], w)
                row += c


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("P", [16, 32, 64, 128])
@pytest.mark.parametrize("D", [64, 128])
def test_append_layouts(g2, fmt, P, D):
    n, table = tables(3, 4)
    cache = Cache(g2, n, 3, P, D, fmt)
    pos = [0, P - 1, P + 3]
    cache.fill(table, pos)
    check_append(g2, cache, [2 * P + 1, 2, 1], pos, table, gather=P < 64)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("ragged", [False, True])
def test_append_one_token_at_a_time(g2, fmt, dtype, ragged):
    """A decode loop: blocks fill up row by row, their scales grow and kept rows are rounded again."""
    n, table = tables(5, 3)
    cache = Cache(g2, n, 2, 16, 64, fmt)
    pos = [0, 7, 15, 16, 31]
    cache.fill(table, pos)
    for step in range(17 if ragged else 5):
        check_append(g2, cache, [1] * 5, [p + step for p in pos] if step < 16 else pos, table, dtype, seed=step, ragged=ragged,
                     gather=step == 0)


@pytest.mark.parametrize("fmt", FMTS)
def test_append_ragged_and_empty(g2, fmt):
    n, table = tables(6, 5)
    cache = Cache(g2, n, 4, 32, 64, fmt)
    pos = [0, 5, 32, 31, 64, 100]
    cache.fill(table, pos)
    check_append(g2, cache, [0, 1, 33, 0, 96, 17], pos, table, "f16")
    check_append(g2, cache, [0, 0, 0, 0, 0, 1], pos, table)


@pytest.mark.parametrize("fmt", FMTS)
def test_append_borders(g2, fmt):
    """Quotients on and beside every rounding border, with a scale that is no power of two."""
    n, table = tables(1, 8)
    cache = Cache(g2, n, 1, 128, 64, fmt)
    gr = grid(fmt)
    s = torch.tensor(1.37, device="cuda") / TOP[fmt]
    mid = ((gr[1:] + gr[:-1]) / 2 * s.double()).float()
    x = torch.cat([mid, torch.nextafter(mid, mid + 1), torch.nextafter(mid, mid - 1)])
    x = torch.cat([x, -x])
    rows = -(-len(x) // 63)
    k = torch.full((rows, 1, 64), 0.0, device="cuda")
    k.view(rows, 64)[:, 0] = s * TOP[fmt]
    k.view(rows, 64)[:, 1:] = torch.cat([x, x.new_zeros(rows * 63 - len(x))]).view(rows, 63)
    check_append(g2, cache, [rows], [0], table, k=k, v=-k)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("size", [0.0, 1e-40, 1e-25, 2.0 ** -64 * 100, 1e-10, 6e4, 3e38])
def test_append_magnitudes(g2, fmt, size):
    n, table = tables(2, 2)
    cache = Cache(g2, n, 2, 16, 64, fmt)
    cache.fill(table, [0, 5])
    k = torch.randn(6, 2, 64, device="cuda", generator=gen(8)).clamp(-1, 1) * size
    check_append(g2, cache, [5, 1], [0, 5], table, k=k, v=k.flip(0))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
def test_append_non_finite(g2, fmt, what):
    """The scale of that page and head becomes NaN and stays so until the page starts anew."""
    n, table = tables(2, 2)
    cache = Cache(g2, n, 3, 16, 64, fmt)
    cache.fill(table, [0, 5])
    k = torch.randn(6, 3, 64, device="cuda", generator=gen(9))
    k[2, 1, 60] = what
    check_append(g2, cache, [3, 3], [0, 5], table, k=k, v=k.flip(0))
    check_append(g2, cache, [1, 1], [3, 8], table)
    check_append(g2, cache, [1, 1], [0, 0], table)
    assert cache.ks[table[:, 0].long()].isfinite().all()


def test_append_again_changes_nothing(g2):
    n, table = tables(3, 3)
    cache = Cache(g2, n, 2, 32, 64, "i8")
    pos = [3, 40, 31]
    cache.fill(table, pos)
    check_append(g2, cache, [9, 3, 2], pos, table)
    was = cache.k.clone(), cache.v.clone(), cache.ks.clone()
    check_append(g2, cache, [9, 3, 2], pos, table)
    assert torch.equal(cache.k, was[0]) and torch.equal(cache.v, was[1]) and same(cache.ks, was[2])


def test_far_pages(g2):
    """Pages whose codes lie past 2^31 bytes."""
    pages, H, P, D = 17000, 16, 128, 64
    k, v = (torch.zeros(pages, H, P, D, dtype=torch.int8, device="cuda") for _ in "kv")
    ks, vs = (torch.zeros(pages, H, device="cuda") for _ in "kv")
    cache = g2.kv8_cache(k, v, ks, vs)
    table = ints([[16999, 3], [16500, 16998]])
    x = torch.randn(200, 2, H, D, device="cuda", generator=gen(10))
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    args = dict(q_start=ints([0, 60, 200]), max_q=140, status=st)
    g2.kv8_append(cache, x[:, 0], x[:, 1], 200, 2, table, 2, ints([0, 0]), row_stride=2 * H * D, **args)
    o = torch.empty_like(x)
    g2.kv8_gather(cache, o[:, 0], o[:, 1], 200, 2, table, 2, ints([0, 0]), row_stride=2 * H * D, **args)
    assert int(st) == 0 and ((o - x).abs() <= x.abs().max() / 254 * 1.001).all()
    out = torch.empty(200, H, D, device="cuda")
    ws = torch.zeros(g2.kv8_attention_workspace(cache, H, 2, 140), dtype=torch.uint8, device="cuda")
    g2.kv8_attention(cache, x[:, 0], out, H, 200, 2, table, 2, ints([60, 140]), ws, ws.numel(), q_stride=2 * H * D, **args)
    for a, b in ((0, 60), (60, 200)):
        q, kk, vv = x[a:b, 0].double(), o[a:b, 0].double(), o[a:b, 1].double()
        s = torch.einsum("qhd,khd->hqk", q, kk) / 8
        s = s.masked_fill(torch.ones(b - a, b - a, device="cuda").triu(1).bool(), -math.inf)
        want = torch.einsum("hqk,khd->qhd", s.softmax(-1), vv)
        assert (out[a:b] - want).norm() <= 2 ** -16 * want.norm()


# ---- attention ----------------------------------------------------------------------------
def model_attention(cache, q, counts, lens, table, scale, skip=()):
    """Results, elementwise bounds without the output's own rounding, and the largest A."""
    Hq, D, P = q.shape[1], cache.D, cache.P
    G = Hq // cache.H
    want, tol, most, row = torch.zeros(q.shape, dtype=torch.double, device="cuda"), None, 0.0, 0
    tol = torch.zeros_like(want)
    for s, (m, n) in enumerate(zip(counts, lens)):
        pages = table[s, :-(-n // P)].long()
        keep = torch.tensor([int(p) not in skip for p in pages], device="cuda").repeat_interleave(P)[:n] if n else None
        pages = torch.where((pages >= 0) & (pages < len(cache.k)), pages, 0)
        if n:
            k, v = ((values(c[pages], cache.fmt) * sc[pages].double()[:, :, None, None]).transpose(0, 1).reshape(cache.H, -1, D)[:, :n]
                    for c, sc in ((cache.k, cache.ks), (cache.v, cache.vs)))
            k, v = (x[:, keep] for x in (k, v))
            at = torch.arange(n, device="cuda")[keep]
        for j in range(m):
            upto = n - m + j + 1
            if upto <= 0 or not (at < upto).any():
                continue
            see = at < upto
            qq = q[row + j].double().view(cache.H, G, D)
            sc = torch.einsum("hgd,hkd->hgk", qq, k[:, see]) * scale
            A = float((torch.einsum("hgd,hkd->hgk", qq.abs(), k[:, see].abs()) * scale).max())
            p = sc.softmax(-1)
            want[row + j] = torch.einsum("hgk,hkd->hgd", p, v[:, see]).reshape(Hq, D)
            size = torch.einsum("hgk,hkd->hgd", p, v[:, see].abs()).reshape(Hq, D)
            vs = cache.vs[pages].double().repeat_interleave(P, 0)[:n][keep][see].T[:, None]
            most_w = (p * vs).amax(-1).reshape(Hq, 1) * TOP[cache.fmt]
            tol[row + j] = (2 ** -17 * A + 2 ** -21 + (upto / 16 + 16) * 2 ** -22) * size + upto * 2 ** -35 * most_w
            most = max(most, A)
        row += m
    return want, tol, most


def check_attention(g2, cache, counts, lens, table, group=1, dtype="f32", seed=5, scale=None, q_size=1.0, ws=None, stream=0,
                    strided=False, ragged=True, skip=(), status=0):
    n, Hq, D = sum(counts), cache.H * group, cache.D
    dt, code = (torch.float32, g2.G2_F32) if dtype == "f32" else (torch.float16, g2.G2_F16)
    q = (torch.randn(n, Hq, D, device="cuda", generator=gen(seed)) * q_size).to(dt)
    pad = 16 if strided else 0
    E = Hq * D
    qb = torch.zeros(n + 1, E + pad, device="cuda", dtype=dt)
    qb[:n, :E] = q.view(n, E)
    ob = torch.full((n + 1, E + 2 * pad), 5.5, device="cuda", dtype=dt)
    starts = [0]
    for c in counts:
        starts.append(starts[-1] + c)
    if ws is None:
        ws = torch.zeros(g2.kv8_attention_workspace(cache.h, Hq, len(counts), max(counts + [1])), dtype=torch.uint8, device="cuda")
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    kw = dict(q_start=ints(starts), max_q=max(counts + [1])) if ragged else {}
    args = (cache.h, qb, ob, Hq, n, len(counts), table, table.shape[1], ints(lens), ws, ws.numel())
    kw.update(scale=scale, q_stride=E + pad if strided else 0, out_stride=E + 2 * pad if strided else 0, dtype=code, status=st, stream=stream)
    torch.cuda.synchronize()
    g2.kv8_attention(*args, **kw)
    torch.cuda.synchronize()
    assert int(st) == status
    out = ob[:n, :E].reshape(n, Hq, D).clone()
    assert (ob[n:] == 5.5).all() and (ob[:, E:] == 5.5).all()
    want, tol, A = model_attention(cache, q, counts, lens, table, D ** -0.5 if scale is None else scale, skip)
    half = torch.finfo(dt).eps / 2
    assert out.isfinite().all()
    err = (out.double() - want).abs()
    # fp16 has no steps below 2^-24
    assert (err <= tol + half * want.abs() + (2 ** -25 if dtype == "f16" else 0)).all()
    if n * Hq > 8:
        assert err.norm() <= ((1 + A) * 2 ** -19 + (half if dtype == "f16" else 0)) * want.norm() + 1e-12
    assert (out[tol == 0] == 0).all()      # rows that see nothing
    g2.kv8_attention(*args, **kw)          # the workspace was left ready, and the bits repeat
    torch.cuda.synchronize()
    assert torch.equal(ob[:n, :E].reshape(n, Hq, D), out)
    return out


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("P", [16, 32, 64, 128])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attention_layouts(g2, fmt, P, D, dtype):
    lens = [1, 15, 16, 17, P, P + 1, 2 * P + 7, 0, 300]
    n, table = tables(len(lens), -(-300 // P))
    cache = Cache(g2, n, 3, P, D, fmt)
    cache.fill(table, lens)
    check_attention(g2, cache, [1] * len(lens), lens, table, dtype=dtype, ragged=False)
    check_attention(g2, cache, [1] * len(lens), lens, table, group=2, dtype=dtype, strided=True)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 8, 12])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_shared_heads(g2, fmt, group, D):
    lens = [70, 1, 200]
    n, table = tables(3, 7)
    cache = Cache(g2, n, 2, 32, D, fmt)
    cache.fill(table, lens)
    check_attention(g2, cache, [1, 1, 1], lens, table, group=group)
    check_attention(g2, cache, [3, 0, 2], lens, table, group=group, dtype="f16")


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("counts,lens", [([5], [5]), ([1, 0, 7, 2], [40, 9, 7, 300]), ([40, 3], [41, 90]), ([4, 9, 2], [2, 0, 1]),
                                         ([17, 130], [500, 130])])
def test_attention_several_rows(g2, fmt, D, counts, lens):
    """Causal rows, some of which see nothing because there are more rows than tokens."""
    n, table = tables(len(lens), 16)
    cache = Cache(g2, n, 2, 32, D, fmt)
    cache.fill(table, lens)
    check_attention(g2, cache, counts, lens, table)
    check_attention(g2, cache, counts, lens, table, group=3, dtype="f16")


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("seqs,heads,most", [(1, 1, 6000), (1, 12, 5001), (2, 3, 20000), (40, 12, 700), (200, 2, 90), (150, 16, 60)])
def test_attention_work_is_shared(g2, fmt, seqs, heads, most):
    """Few long sequences, many short ones: rows split over blocks and blocks that take many rows."""
    g = torch.Generator().manual_seed(seqs)
    lens = torch.randint(0, most + 1, (seqs,), generator=g).tolist()
    lens[-1] = most
    n, table = tables(seqs, -(-most // 64))
    cache = Cache(g2, n, heads, 64, 64, fmt)
    cache.fill(table, lens)
    check_attention(g2, cache, [1] * seqs, lens, table, ragged=False)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("spread", [0.0, 10.0])
@pytest.mark.parametrize("q_size", [0.0, 1e-6, 30.0])
def test_attention_ranges(g2, fmt, spread, q_size):
    """Pages whose scales lie far apart, sharp and flat softmaxes."""
    lens = [333, 64]
    n, table = tables(2, 11)
    cache = Cache(g2, n, 2, 32, 64, fmt)
    cache.fill(table, lens, spread=spread)
    cache.ks.copy_(torch.where(cache.ks.isnan(), cache.ks, cache.ks / (cache.ks * 0 + 2 ** spread)))
    check_attention(g2, cache, [2, 1], lens, table, q_size=q_size)
    check_attention(g2, cache, [2, 1], lens, table, q_size=q_size, scale=0.031)


def test_attention_large_q(g2):
    """Queries past fp16's range keep fp32 accuracy."""
    n, table = tables(1, 4)
    cache = Cache(g2, n, 2, 32, 64, "i8")
    cache.fill(table, [100])
    check_attention(g2, cache, [1], [100], table, q_size=3e5, scale=1e-6)


def attend(g2, cache, q, lens, table, scale):
    """One query row a sequence, fp32."""
    n, Hq, _ = q.shape
    out = torch.empty_like(q)
    ws = torch.zeros(g2.kv8_attention_workspace(cache.h, Hq, n, 1), dtype=torch.uint8, device="cuda")
    g2.kv8_attention(cache.h, q, out, Hq, n, n, table, table.shape[1], ints(lens), ws, ws.numel(), scale=scale)
    return out


@pytest.mark.parametrize("fmt", FMTS)
def test_attention_largest_q(g2, fmt):
    """Queries in fp32's last power of two, 2^127 and above."""
    n, table = tables(1, 4)
    cache = Cache(g2, n, 2, 32, 64, fmt)
    cache.fill(table, [100])
    q = (torch.randn(1, 2, 64, device="cuda", generator=gen(8)) * 1e38).clamp(-3.4e38, 3.4e38)
    q[:, :, 5], q[:, :, 40] = 3.4e38, -(2.0 ** 127)
    out = attend(g2, cache, q, [100], table, 2e-38)
    want, tol, _ = model_attention(cache, q, [1], [100], table, 2e-38)
    assert ((out.double() - want).abs() <= tol + 2 ** -24 * want.abs()).all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("lens", [[100, 33], [9000, 1]])
def test_attention_far_below_zero(g2, fmt, lens):
    """Scores near fp32's least, all of a row the same: its result is the mean of the values."""
    n, table = tables(2, -(-max(lens) // 32))
    cache = Cache(g2, n, 2, 32, 64, fmt)
    cache.fill(table, lens, spread=0.0)
    one = torch.ones(1, device="cuda")
    cache.k.copy_(one.to(torch.int8) if fmt == "i8" else one.to(torch.float8_e4m3fn).view(torch.int8))
    cache.ks.fill_(1e28)
    q = torch.full((2, 2, 64), -1e8, device="cuda")      # 64 of them by 1e28: -6.4e37, in powers of two -9.2e37
    out = attend(g2, cache, q, lens, table, 1.0)
    for s, m in enumerate(lens):
        pages = table[s, :-(-m // 32)].long()
        v = (values(cache.v[pages], fmt) * cache.vs[pages].double()[:, :, None, None]).transpose(0, 1).reshape(2, -1, 64)[:, :m]
        # the scores lose log2 of the V scales, so equal weights need equal scales
        assert (cache.vs[pages] == cache.vs[pages][0, 0]).all()
        assert ((out[s].double() - v.mean(1)).abs() <= (m / 16 + 16) * 2 ** -22 * v.abs().mean(1)).all()


def test_attention_non_finite_scale(g2):
    """A NaN page shows in the rows and heads that see it, and in no other."""
    lens = [100, 100]
    n, table = tables(2, 4)
    cache = Cache(g2, n, 2, 32, 64, "i8")
    cache.fill(table, lens)
    cache.ks[table[0, 1].long(), 1] = math.nan
    cache.vs[table[1, 3].long(), 0] = math.nan
    q = torch.randn(4, 2, 64, device="cuda", generator=gen(6))
    out = torch.empty_like(q)
    ws = torch.zeros(g2.kv8_attention_workspace(cache.h, 2, 2, 2), dtype=torch.uint8, device="cuda")
    g2.kv8_attention(cache.h, q, out, 2, 4, 2, table, 4, ints(lens), ws, ws.numel(), q_start=ints([0, 2, 4]), max_q=2)
    nan = out.isnan().all(-1).cpu().tolist()
    assert nan == [[False, True], [False, True], [True, False], [True, False]]
    assert torch.equal(out.isnan().any(-1), out.isnan().all(-1))


@pytest.mark.parametrize("fmt", FMTS)
def test_bad_pages_and_sequences_are_skipped(g2, fmt):
    """Out-of-range page ids, lengths, positions and counts are reported, and nothing is read or written for them."""
    lens = [100, 100, 100]
    n, table = tables(3, 4)
    cache = Cache(g2, n, 2, 32, 64, fmt)
    cache.fill(table, lens)
    t = table.clone()
    t[0, 1], t[1, 3], t[2, 0] = -1, n, 2 ** 30
    check_attention(g2, cache, [1, 2, 1], lens, t, skip=(-1, n, 2 ** 30), status=-6)
    q = torch.randn(4, 2, 64, device="cuda")
    st, ws = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(g2.kv8_attention_workspace(cache.h, 2, 3, 2), dtype=torch.uint8, device="cuda")
    for ln, qs in (([100, 129, -1], [0, 1, 3, 4]), ([100, 100, 100], [0, 1, 0, 1]), ([100] * 3, [0, 1, 4, 4]), ([100] * 3, [0, 1, 1, 5])):
        st.zero_()
        out = torch.full_like(q, 7.0)
        g2.kv8_attention(cache.h, q, out, 2, 4, 3, table, 4, ints(ln), ws, ws.numel(), q_start=ints(qs), max_q=2, status=st)
        assert int(st) == -6 and out.isfinite().all() and (out[3] == 7).all() and not (out[0] == 7).any()
    before = [x.clone() for x in (cache.k, cache.v, cache.ks, cache.vs)]
    for pos, qs, tb in (([-1, 128, 127], [0, 1, 2, 4], table), ([0, 0, 0], [0, 3, 3, 3], table), ([0, 0, 0], [0, -1, 4, 3], table),
                        ([40, 100, 0], [0, 1, 2, 4], t)):
        st.zero_()
        g2.kv8_append(cache.h, q, q, 4, 3, tb, 4, ints(pos), q_start=ints(qs), max_q=2, status=st)
        o = torch.full_like(q, 7.0)
        g2.kv8_gather(cache.h, o, o.clone(), 4, 3, tb, 4, ints(pos), q_start=ints(qs), max_q=2)
        assert int(st) == -6 and (o == 7).all()
        assert all(same(a, b) if a.is_floating_point() else torch.equal(a, b) for a, b in zip(before, (cache.k, cache.v, cache.ks, cache.vs)))


def test_streams_and_capture(g2):
    """Two streams with a workspace each, and a captured decode step replayed as the lengths grow."""
    lens = [500, 30, 257, 64]
    n, table = tables(4, 9)
    cache = Cache(g2, n, 4, 64, 64, "i8")
    cache.fill(table, lens)
    want = check_attention(g2, cache, [1] * 4, lens, table, seed=7)
    q = torch.randn(4, 4, 64, device="cuda", generator=gen(7))
    size = g2.kv8_attention_workspace(cache.h, 4, 4, 1)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty(30, 4, 4, 64, device="cuda") for _ in streams]
    wss = [torch.zeros(size, dtype=torch.uint8, device="cuda") for _ in streams]
    L = ints(lens)
    torch.cuda.synchronize()
    for i in range(30):
        for st, o, w in zip(streams, outs, wss):
            g2.kv8_attention(cache.h, q, o[i], 4, 4, 4, table, 9, L, w, size, stream=st.cuda_stream)
    torch.cuda.synchronize()
    assert all((o == want).all() for o in outs)
    # append one token, then attend; positions and lengths live on the device
    kv, out, pos = torch.empty(4, 2, 256, device="cuda"), torch.empty(4, 4, 64, device="cuda"), ints(lens)
    one = torch.ones(4, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s = torch.cuda.current_stream().cuda_stream
        g2.kv8_append(cache.h, kv[:, 0], kv[:, 1], 4, 4, table, 9, pos, row_stride=512, stream=s)
        g2.kv8_attention(cache.h, q, out, 4, 4, 4, table, 9, L, wss[0], size, stream=s)
    for step in range(20):
        kv.copy_(torch.randn(4, 2, 256, device="cuda", generator=gen(100 + step)))
        L.add_(one)
        graph.replay()
        pos.add_(one)
        torch.cuda.synchronize()
    now = [v + 20 for v in lens]
    assert torch.equal(out, check_attention(g2, cache, [1] * 4, now, table, seed=7))
