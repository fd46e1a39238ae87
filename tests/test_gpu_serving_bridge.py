"""The serving operators through the torch bridge with every setting that ``arke_b200.ops`` has: a compiled decode step
with settings per request can be written with it."""
import pytest
import torch


def _bridge():
    from arke_b200 import bridge, ops
    assert bridge.register_ops()
    return torch.ops.arke, ops


def test_schemas_carry_the_settings():
    a, _ = _bridge()
    names = lambda op: [x.name for x in op.default._schema.arguments]  # noqa: E731
    assert {"cu_q", "positions"} <= set(names(a.qkv_rope_paged_append))
    assert {"cu_q", "shared_prefix", "causal", "softmax_scale", "max_new"} <= set(names(a.paged_gqa_fwd))
    for op in (a.sample_tokens, a.sample_tokens_logprob):
        assert {"temperature_rows", "top_k_rows", "top_p_rows", "min_p_rows"} <= set(names(op))


@pytest.fixture
def step():
    g = torch.Generator(device="cuda").manual_seed(1)
    Hq, Hkv, D, page = 4, 2, 64, 16
    k, v = (torch.randn(6, Hkv, page, D, generator=g, device="cuda").half() for _ in range(2))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    return {"k": k, "v": v, "table": torch.arange(6, dtype=torch.int32, device="cuda").view(2, 3), "lens": i32([40, 23]), "cu": i32([0, 1, 3]),
            "pos": i32([7, 0, 47]), "qkv": torch.randn(4, (Hq + 2 * Hkv) * D, generator=g, device="cuda").half(), "Hq": Hq,
            "cos": torch.rand(48, D // 2, generator=g, device="cuda"), "sin": torch.rand(48, D // 2, generator=g, device="cuda"),
            "x": torch.randn(3, 999, generator=g, device="cuda"), "u": torch.rand(3, generator=g, device="cuda"),
            "t": torch.tensor([0.0, 0.7, 1.3], device="cuda"), "tk": i32([0, 5, 40]), "tp": torch.tensor([1.0, 0.9, 0.5], device="cuda"),
            "mp": torch.tensor([0.0, 0.1, 0.01], device="cuda")}


@pytest.mark.gpu
@pytest.mark.parametrize("cu", [True, False])
@pytest.mark.parametrize("pos", [True, False])
def test_append(step, cu, pos):
    a, ops = _bridge()
    s = step
    qkv = s["qkv"] if cu else s["qkv"][:2]
    c, p = (s["cu"] if cu else None), (torch.cat([s["pos"], s["pos"][:1]])[:qkv.shape[0]].contiguous() if pos else None)
    k2, v2 = s["k"].clone(), s["v"].clone()
    q = a.qkv_rope_paged_append(qkv, s["cos"], s["sin"], s["k"], s["v"], s["table"], s["lens"], c, s["Hq"], p)
    want = ops.qkv_rope_paged_append(qkv, s["cos"], s["sin"], k2, v2, s["table"], s["lens"], s["Hq"], cu_q=c, positions=p)
    assert torch.equal(q, want) and torch.equal(k2, s["k"]) and torch.equal(v2, s["v"])


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(), dict(causal=False), dict(softmax_scale=0.3), dict(max_new=2), dict(causal=False, softmax_scale=0.05)], ids=str)
@pytest.mark.parametrize("cu", [True, False])
def test_attention(step, kw, cu):
    a, ops = _bridge()
    s = step
    q = s["qkv"].view(4, -1, 64)[:, :s["Hq"]]
    c = s["cu"] if cu else None
    o, lse = a.paged_gqa_fwd(q, s["k"], s["v"], s["table"], s["lens"], c, 16, **kw)
    o2, lse2 = ops.paged_gqa_fwd(q, s["k"], s["v"], s["table"], s["lens"], cu_q=c, shared_prefix=16, **kw)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)


@pytest.mark.gpu
def test_sampling_with_settings_of_each_row(step):
    a, ops = _bridge()
    s = step
    rows = dict(temperature_rows=s["t"], top_k_rows=s["tk"], top_p_rows=s["tp"], min_p_rows=s["mp"])
    want, lp = ops.sample_tokens(s["x"], s["u"], s["t"], s["tk"], s["tp"], s["mp"], return_logprob=True)
    assert torch.equal(a.sample_tokens(s["x"], s["u"], **rows), want)
    token, logprob = a.sample_tokens_logprob(s["x"], s["u"], **rows)
    assert torch.equal(token, want) and torch.equal(logprob, lp)
    # one setting per row, the others for all
    token, logprob = a.sample_tokens_logprob(s["x"], s["u"], 0.8, 0, 0.9, 0.0, top_k_rows=s["tk"])
    want, lp = ops.sample_tokens(s["x"], s["u"], 0.8, s["tk"], 0.9, 0.0, return_logprob=True)
    assert torch.equal(token, want) and torch.equal(logprob, lp)


@pytest.mark.gpu
def test_a_decode_step_is_one_graph(step):
    """Traced without a break, and the same numbers as without tracing."""
    a, ops = _bridge()
    s = step

    def decode(qkv, k, v, t, tk):
        q = a.qkv_rope_paged_append(qkv, s["cos"], s["sin"], k, v, s["table"], s["lens"], None, s["Hq"])
        o, _ = a.paged_gqa_fwd(q, k, v, s["table"], s["lens"], None, 0, softmax_scale=0.2)
        logits = o.float().reshape(2, -1)
        return a.sample_tokens_logprob(logits, s["u"][:2], temperature_rows=t, top_k_rows=tk)

    k2, v2 = s["k"].clone(), s["v"].clone()
    t, tk = s["t"][1:].contiguous(), s["tk"][1:].contiguous()
    want = decode(s["qkv"][:2], k2, v2, t, tk)
    got = torch.compile(decode, backend="eager", fullgraph=True)(s["qkv"][:2], s["k"], s["v"], t, tk)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(s["k"], k2) and torch.equal(s["v"], v2)
