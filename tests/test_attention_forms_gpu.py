"""Every form that the attention's host rules can choose, at every padded width, both types, with and without a causal mask, a key mask, a bias and a negative
scale: out, lse and all gradients against the 64-bit definition."""
import random

import pytest
import torch

from tf_repos_amd import capi
from tests.seq_util import AttentionCase

pytestmark = pytest.mark.gpu
ALL = ("out", "lse", "dq", "dk", "dv", "db")


def run(case, dev):
    d = case.to(dev)
    capi.check(case.forward(d))
    capi.check(case.backward(d))
    torch.cuda.synchronize()
    assert d["status"].tolist() == [0, 0]
    case.check(d, ALL)


def lengths(seed, n, q, k):
    r = random.Random(seed)
    return [q] + [r.randint(0, q) for _ in range(n - 1)], [k] + [0 if r.random() < 0.1 else r.randint(1, k) for _ in range(n - 1)]


# sizes for which the rules choose: rows of queries and keys in blocks of 128 shared by four waves; blocks of 32 whose waves split the other side; a wave
# for each 32 rows; and one query a segment (forward split over the keys)
FORMS = {"rows": (16, 200, 300, 8), "split": (3, 60, 200, 2), "solo": (300, 20, 60, 4), "few": (5, 2, 700, 2)}


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [24, 64, 72, 128])
@pytest.mark.parametrize("form", sorted(FORMS))
@pytest.mark.parametrize("causal", [False, True])
def test_every_form(form, dim, dtype, causal, dev):
    n, q, k, heads = FORMS[form]
    q, k = lengths(n + dim, n, q, k)
    run(AttentionCase(dtype, q, k, heads, heads, dim, causal=causal, boundaries=[-90, -30, -5, -1, 0, 1, 40], q_start=[max(0, b - a) for a, b in zip(q, k)],
                      keep=lambda j: j % 11 != 3, seed=60 + dim), dev)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [16, 64, 128])
@pytest.mark.parametrize("form", sorted(FORMS))
def test_negative_scale(form, dim, dtype, dev):
    n, q, k, heads = FORMS[form]
    q, k = lengths(n, n, q, k)
    run(AttentionCase(dtype, q, k, heads, heads, dim, causal=form == "rows", boundaries=[-3, 0] if dim == 64 else None, scale=-0.3, seed=61), dev)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [40, 64, 128])
def test_rows_of_shared_heads(dim, dtype, dev):
    """Blocks of 128 rows on both sides with several query heads a key head."""
    q, k = lengths(62, 30, 200, 300)
    run(AttentionCase(dtype, q, k, 16, 8, dim, causal=True, boundaries=[-33, -2, 0], q_start=[max(0, b - a) for a, b in zip(q, k)], seed=62), dev)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("form", sorted(FORMS))
def test_a_scale_of_zero_weighs_every_key_alike(form, dtype, dev):
    n, q, k, heads = FORMS[form]
    q, k = lengths(n + 1, n, q, k)
    run(AttentionCase(dtype, q, k, heads, heads, 32, scale=0.0, seed=63), dev)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("form", sorted(FORMS))
def test_without_the_optional_outputs(form, dtype, dev):
    """No lse from a forward alone, no bias gradient from a backward with a bias: the rest is the same, bit by bit."""
    n, q, k, heads = FORMS[form]
    q, k = lengths(n + 2, n, q, k)
    case = AttentionCase(dtype, q, k, heads, heads, 64, causal=True, boundaries=[-9, 0], q_start=[max(0, b - a) for a, b in zip(q, k)], seed=64)
    full, part = case.to(dev), case.to(dev)
    capi.check(case.forward(full))
    capi.check(case.backward(full))
    capi.check(case.forward(part, lse=False))
    assert torch.all(part["lse"] == 7.0)
    part["lse"].copy_(full["lse"])
    a, p = case.describe(), capi.ptr
    capi.check(capi.lib().dctr_cross_attention_bwd(*case.ins(a, part), p(part["out"]), case.q_ld, p(part["lse"]), p(part["do"]), case.q_ld, p(part["dq"]), case.q_ld,
                                                   p(part["dk"]), case.k_ld, p(part["dv"]), case.v_ld, None, p(part["ws1"]), part["bytes1"], capi.current_stream()))
    torch.cuda.synchronize()
    for n in ("out", "dq", "dk", "dv"):
        assert torch.equal(full[n], part[n]), n


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_two_calls_at_once(dtype, dev):
    """Two streams, a workspace each, with other calls between: the results of the calls alone."""
    cases = [AttentionCase(dtype, *lengths(65 + i, *FORMS[f][:3]), FORMS[f][3], FORMS[f][3], 64, causal=True, boundaries=[-9, 0], seed=65 + i)
             for i, f in enumerate(("rows", "few"))]
    alone = []
    for c in cases:
        d = c.to(dev)
        capi.check(c.forward(d))
        capi.check(c.backward(d))
        alone.append(d)
    both, streams = [c.to(dev) for c in cases], [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        for c, d, s in zip(cases, both, streams):
            capi.check(c.forward(d, stream=capi.ptr(s.cuda_stream)))
            capi.check(c.backward(d, stream=capi.ptr(s.cuda_stream)))
    torch.cuda.synchronize()
    for x, y in zip(alone, both):
        for n in ALL:
            assert torch.equal(x[n], y[n]), n


@pytest.mark.parametrize("dim", [24, 64])
@pytest.mark.parametrize("form", ["split", "solo"])
@pytest.mark.parametrize("causal", [False, True])
def test_small_gradients_are_rounded_once(form, dim, causal, dev):
    """bf16 gradients of few or short lists are as far off as their own rounding makes them: an error spread over a step of 2^-7 of the power of two below a
    value has the root mean square 2^-7 / sqrt(12) = 0.00226 of that, and less of the value (0.0017 of normal ones).  Weights rounded before them make
    sqrt(2) times the 0.0017, 0.00235."""
    n, q, k, heads = FORMS[form]
    q, k = lengths(n + dim, n, q, k)
    case = AttentionCase("bf16", q, k, heads, heads, dim, causal=causal, boundaries=[-5, 0], q_start=[max(0, b - a) for a, b in zip(q, k)], seed=70)
    d, ref = case.to(dev), case.reference()
    capi.check(case.forward(d))
    capi.check(case.backward(d))
    for name, rows in (("dq", case.nq), ("dk", case.nk), ("dv", case.nk)):
        got = d[name][:rows, :heads * dim].cpu().double().view(rows, heads, dim)
        off = ((got - ref[name][0]).norm() / ref[name][0].norm()).item()
        assert off <= 2.0 ** -7 / 12 ** 0.5, (name, off)
