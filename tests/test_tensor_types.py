"""The Python calls of the 4-bit, 8-bit-cache and logit-rule operators refuse tensors
whose elements have the right size but another meaning (bf16 for fp16, int32 for fp32),
on the CPU: the check comes before the library is called."""
import pytest

torch = pytest.importorskip("torch")
import gpt2b200 as g2  # noqa: E402
from test_operator_args import A, CALLS, ARG, cache, code  # noqa: E402

B, I = torch.zeros(4096, dtype=torch.bfloat16), torch.zeros(4096, dtype=torch.int32)


def test_weights_and_rows():
    assert code(g2.q4_pack, B, A, 16, 64, 32, dict(dtype=g2.G2_F16)) == ARG
    assert code(g2.q4_pack, I, A, 16, 64, 32, {}) == ARG
    assert code(g2.q4_unpack, A, I, 16, 64, 32) == ARG
    for bad in (dict(x=B, dtype=1), dict(y=B, dtype=1), dict(residual=B, dtype=1), dict(x=I), dict(bias=I), dict(ln_gamma=I, ln_beta=A),
                dict(ln_gamma=A, ln_beta=I)):
        k = dict(bad)
        assert "torch" in str(pytest.raises(g2.G2Error, g2.matvec_q4, k.pop("x", A), A, k.pop("y", A), 1, 16, 64, 32, **k).value), bad


@pytest.mark.parametrize("name", CALLS)
def test_cache_rows(name):
    for bad in (dict(a=B, dtype=1), dict(b=B, dtype=1), dict(a=I), dict(b=I)):
        with pytest.raises(g2.G2Error, match="torch"):
            CALLS[name](cache(), dict(bad))


def test_cache_scales_and_rules():
    k, s = torch.zeros(4, 2, 16, 64, dtype=torch.int8), torch.zeros(4, 2)
    for bad in ((k, k, s.int(), s), (k, k, s, s.int())):
        assert code(g2.kv8_cache, *bad) == ARG
    for bad in (dict(rep_penalty=I), dict(presence=I), dict(frequency=I), dict(bias=I, bias_ids=I)):
        with pytest.raises(g2.G2Error, match="torch"):
            g2.logit_rules(**bad)
    with pytest.raises(g2.G2Error, match="torch"):
        g2.process_logits(I, I, 1, 64, g2.logit_rules())


def test_rules_are_contiguous():
    """The rules' lengths are those of the tensors, so every other element would be read as the next one."""
    for bad in (dict(ctx=I[::2]), dict(mask=I[::2]), dict(bias=torch.zeros(64)[::2], bias_ids=I[:32]), dict(rep_penalty=torch.zeros(64)[::2])):
        with pytest.raises(g2.G2Error, match="contiguous"):
            g2.logit_rules(**bad)
