"""GPU: sampling where the decision falls into a long tail of tiny weights, against 64-bit sums.

A weight may be off by 2^-42 of itself and by 2^-85 of the largest one (2^-60 where top-p looks for its border), so
running sums inside a tail are off by that much of the tail, not of the whole; at u = 0 the first kept token whose 64-bit
weight is not zero is chosen, however small that weight is."""
import math

import numpy as np
import pytest
import torch

from oracle import serving as oracle

pytestmark = pytest.mark.gpu
LN2 = math.log(2.0)


def _ops():
    from arke_b200 import ops
    return ops


def rows(v, n, dtype=torch.float32):
    return torch.full((n,), v, dtype=dtype, device="cuda")


def tail(V, level, peak=None, inside=()):
    """All logits at -level ln 2 but for a 0 at `peak` (the last) and the given (index, level) pairs."""
    x = torch.full((V,), -level * LN2, dtype=torch.float32)
    x[V - 1 if peak is None else peak] = 0.0
    for i, at in inside:
        x[i] = -at * LN2
    return x


def expected(x, us, order):
    """Tokens that running sums in extended precision choose among `order` (ascending indexes), None where the border is
    closer than what the sums may be off."""
    w = np.exp(x.double().numpy()[order]).astype(np.longdouble)
    c = np.cumsum(w)
    out = []
    for u in us:
        t = np.longdouble(u) * c[-1]
        j = int(np.searchsorted(c, t, side="right"))
        near = np.abs(c[max(0, j - 1):j + 1] - t).min()
        out.append(int(order[j]) if near > t * 2.0 ** -41 + len(order) * np.longdouble(2.0) ** -84 or u == 0 else None)
    return out


US = [0.0, 2.0 ** -40, 2.0 ** -32, 2.0 ** -30, 3 * 2.0 ** -29, 2.0 ** -27, 2.0 ** -25, 5 * 2.0 ** -27, 2.0 ** -24, 0.25, 1 - 2.0 ** -24]
TAILS = [(1 << 20, 44.1, ()), (128256, 45.1, ()), (128256, 43.0, ((50000, 24.0),)), (128256, 46.0, ((70000, 24.0), (3, 40.0))),
         (50257, 47.5, ((20000, 25.5),)), (1 << 20, 47.9, ())]


@pytest.mark.parametrize("V, level, inside", TAILS, ids=lambda v: str(v))
@pytest.mark.parametrize("how", ["plain", "plain rows", "top_k", "min_p"])
def test_borders_inside_a_tail(V, level, inside, how):
    x = tail(V, level, inside=inside)
    n = len(US)
    order = np.arange(V)
    kw = {}
    if how == "plain rows":
        kw = dict(temperature=rows(1.0, n), top_k=rows(0, n, torch.int32), top_p=rows(1.0, n), min_p=rows(0.0, n))
    elif how == "top_k":                       # the last third of the tail's equals stays out
        k = V - V // 3
        kw = dict(top_k=k)
        order = np.sort(np.lexsort((order, -x.double().numpy()))[:k])
    elif how == "min_p":                       # everything stays in, and has to be compared
        kw = dict(min_p=2.0 ** -50)
    want = expected(x, US, order)
    got = _ops().sample_tokens(x.cuda().expand(n, V).contiguous(), torch.tensor(US).cuda(), **kw).cpu().tolist()
    sure = [i for i in range(n) if want[i] is not None]
    assert len(sure) >= n - 2 and [got[i] for i in sure] == [want[i] for i in sure]


@pytest.mark.parametrize("V, level, dt", [(1 << 17, 38.4, torch.float32), (1 << 17, 37.0, torch.bfloat16), (1 << 18, 39.4, torch.float32),
                                          (40000, 36.2, torch.float16)])
def test_top_p_border_inside_a_tail(V, level, dt):
    """All but 2^-24 or 2^-23 of the whole stays: that cuts a tail of equal weights after a number of tokens that sums in
    extended precision say; the last of them is what u = 1 chooses."""
    x = tail(V, level, peak=0).to(dt)
    w = np.exp(x.double().numpy()).astype(np.longdouble)
    before = np.cumsum(w) - w
    for p in (1 - 2.0 ** -24, 1 - 2.0 ** -23):
        t = np.longdouble(p) * w.sum()
        last = int((before < t).sum()) - 1
        # the peak's weight is exact; V weights off by 2^-60 each, and by 2^-42 of the tail
        assert np.abs(before - t).min() > V * np.longdouble(2.0) ** -60 + (w.sum() - 1) * 2.0 ** -42, "the input has no clear border"
        for extra in (dict(), dict(top_k=V - 1)):
            if extra:
                z = w[:-1].sum()
                t2 = np.longdouble(p) * z
                last = int((before[:-1] < t2).sum()) - 1
                assert np.abs(before[:-1] - t2).min() > V * np.longdouble(2.0) ** -60 + (z - 1) * 2.0 ** -42
            token = _ops().sample_tokens(x.cuda()[None], torch.ones(1).cuda(), top_p=p, **extra)
            assert int(token[0]) == last


FIRST = [dict(top_k=3000), dict(top_p=1 - 2.0 ** -24), dict(top_k=2500, top_p=0.9), dict(top_k=3000, min_p=1e-30)]


@pytest.mark.parametrize("f", FIRST, ids=str)
@pytest.mark.parametrize("t", [1.0, 0.5, 3.0])
def test_the_number_zero_chooses_the_first_kept_token(f, t):
    low = torch.finfo(torch.float32).min
    V = 4000
    x = torch.randn(8, V, generator=torch.Generator().manual_seed(1))
    x[:, V - 9] = 9.0
    x[0, :7] = -300.0
    x[1, :7], x[1, 7] = low, -200.0
    x[2, :5] = -math.inf
    x[3, :2000] = -700.0 * t + 9.0               # a 64-bit weight of 1e-304
    x[4, :2000], x[4, 2000:3000] = -760.0 * t + 9.0, -744.0 * t + 9.0      # one of 0, and one that is not
    x[5] = low
    x[5, 3111] = 1.0
    x[6] = 2.5
    x[7, :3999] = -40.0
    got = _ops().sample_tokens(x.cuda(), torch.zeros(8).cuda(), temperature=t, **f).cpu()
    p32, m32 = float(torch.tensor(f.get("top_p", 1.0))), float(torch.tensor(f.get("min_p", 0.0)))
    want = [oracle.sample(r.numpy(), 0.0, t, f.get("top_k", 0), p32, m32)[0] for r in x]
    assert got.tolist() == want


@pytest.mark.parametrize("V, level", [(4096, 60.0), (128256, 49.5), (1 << 20, 49.5), (50257, 300.0)])
@pytest.mark.parametrize("how", ["numbers", "rows", "many rows"])
def test_small_numbers_in_front_of_a_peak(V, level, how):
    """No filter, all the weight in the last token, and a number that falls into the tail in front of it: u = 0, and the
    middle of the tail's share, which is 2^-30 of the whole at most and far from every border."""
    n = 300 if how == "many rows" else 2                    # the kernel for batches without filters starts at some 40 rows
    x = tail(V, level)
    w = math.exp(float(x[0]))
    middle = (V // 2 + 0.5) * w                            # of a whole that is 1 to 2^-29
    u = torch.tensor([0.0, middle], dtype=torch.float32)
    j = expected(x, u.tolist(), np.arange(V))
    kw = {}
    if how == "rows":
        kw = dict(temperature=rows(1.0, n), top_k=rows(0, n, torch.int32), top_p=rows(1.0, n), min_p=rows(0.0, n))
    us = u.cuda().repeat((n + 1) // 2)[:n]
    got = _ops().sample_tokens(x.cuda().expand(n, V).contiguous(), us, **kw).cpu()
    assert (got[0::2] == 0).all()
    if middle >= V * 2.0 ** -80:                            # within what running sums resolve
        assert j[1] is not None and (got[1::2] == j[1]).all()


@pytest.mark.parametrize("n", [4, 400])
@pytest.mark.parametrize("f", [dict(), dict(top_k=999), dict(top_p=0.999999)], ids=str)
def test_min_p_of_one_keeps_what_64_bits_cannot_tell_from_the_largest(n, f):
    """At a temperature of 1e30 every weight is 1 in 64 bits, and 1 >= min_p: the same with and without other filters."""
    V = 1000
    x = torch.randn(V, generator=torch.Generator().manual_seed(1))
    order = np.arange(V)
    kept = f.get("top_k", math.ceil(float(torch.tensor(f.get("top_p", 1.0))) * V))      # of equal weights
    order = np.sort(np.lexsort((order, -x.double().numpy()))[:kept])
    u = (torch.arange(n) + 0.25) / n
    got = _ops().sample_tokens(x.cuda().expand(n, V).contiguous(), u.cuda(), temperature=1e30, min_p=1.0, **f).cpu().tolist()
    assert got == [int(order[int(float(v) * len(order))]) for v in u]
