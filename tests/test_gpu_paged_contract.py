"""GPU: what paged attention promises beyond its results — broken tables, padded batches, the bound of its error — against
64-bit restatements."""
import pytest
import torch

from oracle import serving as oracle
from test_gpu_paged import ATTEND, TILES, _i32, _ops, make_cache, o_tolerance, prefix_units, to_gpu  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new, ctx, Hq, Hkv", [(300, 300, 8, 2), (300, 900, 8, 2), (520, 520, 4, 2), (9, 300, 8, 2), (1, 300, 4, 4)])
@pytest.mark.parametrize("where", ["last", "middle"])
def test_rows_that_see_a_missing_page_are_nan(new, ctx, Hq, Hkv, where):
    """Of a sequence whose rows make several units of 256 those that see the page are NaN; the others are NaN or right, as
    is said of them; the other sequences are right."""
    D, page, dt, lens = 64, 16, torch.bfloat16, [ctx, 40]
    ops = _ops()
    k, v, table = make_cache(lens, Hkv, D, page, dt, "hnd", 5)
    q = torch.randn(new + 1, Hq, D, generator=torch.Generator().manual_seed(2)).to(dt)
    cu = [0, new, new + 1]
    o64, lse64 = oracle.paged_attention(q, k, v, table, lens, cu)
    bad_page = -(-ctx // page) - 1 if where == "last" else -(-ctx // page) // 2
    broken = table.clone()
    broken[0, bad_page] = k.shape[0] + 7
    o, lse = ops.paged_gqa_fwd(q.cuda(), to_gpu(k), to_gpu(v), broken.cuda(), _i32(lens).cuda(), cu_q=_i32(cu).cuda())
    assert ops.kernel_status() == 8 and ops.kernel_status() == 0
    o, lse = o.cpu(), lse.cpu()
    sees = torch.arange(ctx - new, ctx) >= bad_page * page
    assert torch.isnan(o[:new][sees]).all() and torch.isnan(lse[:new][sees]).all()
    big = v.double()[torch.isfinite(v)].abs().max()
    right = (o.double() - o64).abs() <= o_tolerance(o64, v, dt) + torch.finfo(dt).eps / 2 * big
    gone = torch.isnan(o)
    assert (gone[:new][~sees] | right[:new][~sees]).all() and right[new:].all() and torch.isfinite(lse[new:]).all()
    assert torch.equal(gone.all(2), gone.any(2)) and torch.equal(torch.isnan(lse), gone.all(2))      # a row is NaN as a whole


PADDED = [  # new tokens of each slot, lengths, heads, head_dim, page
    ([0] * 300 + [200] + [0] * 99, [40] * 300 + [333] + [7] * 99, 8, 2, 64, 16),          # one prompt, 399 empty slots
    ([0] * 20 + [70] + [0] * 60 + [1, 1, 3] + [0] * 50, [5] * 20 + [70] + [0] * 60 + [90, 31, 3] + [64] * 50, 4, 4, 128, 32),
    ([64] + [0] * 64, [500] + [0] * 64, 8, 1, 64, 8),
    ([0] * 700, [9] * 700, 4, 2, 64, 16),                                                  # nobody has a token
    ([0] * 9 + [3, 1], [20] * 9 + [300, 2], 8, 2, 64, 16),                                 # fewer rows than a tile wants
]


@pytest.mark.parametrize("case", PADDED, ids=lambda c: f"{sum(c[0])}tok{len(c[0])}slots")
@pytest.mark.parametrize("tag", ["bf16", "f16"])
@pytest.mark.parametrize("prefix", [0, 32])
@pytest.mark.parametrize("told", ["nothing", "the longest", "too much", "too little"])
def test_more_empty_sequences_than_tokens(case, tag, prefix, told):
    """A batch of fixed slots, most without a token: the same rows as without the empty ones, rows behind the last are 0,
    whatever the caller says of the longest sequence."""
    new, lens, Hq, Hkv, D, page = case
    if prefix:
        lens = [n + prefix for n in lens]
    dt = {"bf16": torch.bfloat16, "f16": torch.float16}[tag]
    ops = _ops()
    k, v, table = make_cache(lens, Hkv, D, page, dt, "hnd", 9, prefix)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    T = cu[-1] + 3
    q = (torch.randn(T, Hq, D, generator=torch.Generator().manual_seed(3)) * 1.5).to(dt)
    with ops.options(paged_prefix_kb=1):
        o, lse = ops.paged_gqa_fwd(q.cuda(), k.cuda(), v.cuda(), table.cuda(), _i32(lens).cuda(), cu_q=_i32(cu).cuda(), shared_prefix=prefix,
                                   max_new={"nothing": 0, "the longest": max(new), "too much": 1 << 30, "too little": 1}[told])
    o64, lse64 = oracle.paged_attention(q, k, v, table, lens, cu, prefix)
    assert within_weights(o, o64, q, k, v, table, lens, cu, prefix, True)
    seen = torch.isfinite(lse64)
    assert torch.equal(torch.isfinite(lse.cpu()), seen) and (o.cpu()[~seen] == 0).all() and not seen[cu[-1]:].any()
    assert ((lse.cpu().double() - lse64)[seen].abs() <= 2.0 ** -16 + 2.0 ** -23 * lse64[seen].abs()).all()
    assert ops.kernel_status() == 0


def within_weights(o, o64, q, k, v, table, lens, cu, prefix, causal):
    """Half a step of the result; and of the weights, which may be rounded to 16 bits before they meet the values, half a
    step of each (of 2^-25 at least where f16 has no normal numbers; the largest is 1 or more), and 2^-15 of each for
    scores and sums in fp32 (a score below 2^6 is off by 2^-17, its weight and their sum by 2^-16 at most): the error of
    a column is that share of sum_j p_j |v_j|, which is the same attention over |v|."""
    dt = q.dtype
    mean, _ = oracle.paged_attention(q, k, v.abs(), table, lens, cu, prefix, causal)
    eps = torch.finfo(dt).eps
    tol = eps / 2 * o64.abs() + (eps / 2 + 2.0 ** -15) * mean
    if dt == torch.float16:
        tol = tol + max(lens) * 2.0 ** -25 * v.double()[torch.isfinite(v)].abs().max()
    return ((o.cpu().double() - o64).abs() <= tol).all()


@pytest.mark.parametrize("G", [1, 4, 7])
def test_offsets_and_the_longest_sequence_choose_the_same_kernels_as_a_uniform_batch(G):
    """Two sequences of 30 tokens: with cu_q and their length the call does what it does without cu_q, bit for bit."""
    Hkv, D, page, dt, lens = 2, 64, 16, torch.bfloat16, [500, 333]
    ops = _ops()
    k, v, table = make_cache(lens, Hkv, D, page, dt, "hnd", 4)
    q = torch.randn(60, Hkv * G, D, generator=torch.Generator().manual_seed(8)).to(dt).cuda()
    args = (q, k.cuda(), v.cuda(), table.cuda(), _i32(lens).cuda())
    o, lse = ops.paged_gqa_fwd(*args)
    o2, lse2 = ops.paged_gqa_fwd(*args, cu_q=_i32([0, 30, 60]).cuda(), max_new=30)
    assert torch.equal(o, o2) and torch.equal(lse, lse2) and ops.kernel_status() == 0


def test_refusals_of_the_longest_sequence():
    from arke_b200 import _lib
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16, device="cuda")
    table, lens = torch.zeros(2, 2, dtype=torch.int32, device="cuda"), _i32([5, 6]).cuda()
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    for bad in (-1, 1 << 31):
        with pytest.raises(_lib.ArkeB200Error):
            _ops().paged_gqa_fwd(q, k, k, table, lens, max_new=bad)


@pytest.mark.parametrize("case", ATTEND + TILES, ids=lambda c: f"{len(c[0])}seq{sum(c[0])}tok{c[2]}/{c[3]}x{c[4]}p{c[5]}s{c[7]}")
@pytest.mark.parametrize("tag", ["bf16", "f16"])
def test_error_is_within_the_weights_rounding(case, tag, prefix_units):
    """Every column within what the rounding of the weights can move it, not only within what it moves the largest value."""
    new, lens, Hq, Hkv, D, page, layout, prefix, causal = case
    if prefix == 0 and prefix_units == "merged":
        pytest.skip("no prefix")
    dt = {"bf16": torch.bfloat16, "f16": torch.float16}[tag]
    k, v, table = make_cache(lens, Hkv, D, page, dt, layout, len(new) * 5 + D, prefix)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    q = (torch.randn(cu[-1], Hq, D, generator=torch.Generator().manual_seed(12)) * 1.5).to(dt)
    o64, _ = oracle.paged_attention(q, k, v, table, lens, cu, prefix, causal)
    args = (q.cuda(), to_gpu(k), to_gpu(v), table.cuda(), _i32(lens).cuda())
    for max_new in (0, max(new)):
        o, _ = _ops().paged_gqa_fwd(*args, cu_q=_i32(cu).cuda(), shared_prefix=prefix, causal=causal, max_new=max_new)
        assert within_weights(o, o64, q, k, v, table, lens, cu, prefix, causal)
    assert _ops().kernel_status() == 0


def test_error_of_long_sequences_is_within_the_weights_rounding():
    """Thousands of keys, where the result is small beside the largest value: tiles in parts, and tiles beside streamed keys."""
    Hq, Hkv, D, page, dt = 8, 2, 64, 32, torch.bfloat16
    g = torch.Generator().manual_seed(7)
    for new, lens, prefix in [([40, 3], [5000, 3000], 0), ([1] * 24, [2048 + 100 * (b + 1) for b in range(24)], 2048)]:
        k, v, table = make_cache(lens, Hkv, D, page, dt, "hnd", 13, prefix)
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        q = (torch.randn(cu[-1], Hq, D, generator=g) * 1.5).to(dt)
        o64, _ = oracle.paged_attention(q, k, v, table, lens, cu, prefix)
        with _ops().options(paged_prefix_kb=1):
            o, _ = _ops().paged_gqa_fwd(q.cuda(), k.cuda(), v.cuda(), table.cuda(), _i32(lens).cuda(), cu_q=_i32(cu).cuda(),
                                        shared_prefix=prefix, max_new=max(new))
        assert within_weights(o, o64, q, k, v, table, lens, cu, prefix, True)


SHORTER = [  # new, lens, Hq, Hkv, D, page, shared prefix: nobody is as long as the prefix
    ([1, 1, 2], [50, 20, 7], 4, 2, 64, 16, 96),
    ([1] * 24, [100 + 13 * i for i in range(24)], 8, 2, 128, 32, 900),
    ([40, 3], [300, 170], 8, 2, 64, 64, 640),
    ([1, 5], [0, 3], 4, 4, 128, 8, 128),
    ([60, 0, 60], [130, 0, 129], 4, 2, 128, 16, 2048),
    ([300], [310], 4, 2, 64, 16, 1024),
    ([2] * 9, [33] * 9, 3, 3, 64, 24, 480),                 # pages that are not for the tiles
    ([1, 0, 1], [40, 0, 60], 4, 2, 64, 16, 256),            # the slot without a token claims a length, see below
]


@pytest.mark.parametrize("case", SHORTER, ids=lambda c: f"{sum(c[0])}tok{len(c[0])}seq{c[4]}p{c[5]}s{c[6]}")
@pytest.mark.parametrize("tag", ["bf16", "f16"])
@pytest.mark.parametrize("causal", [True, False])
def test_sequences_shorter_than_the_shared_prefix(case, tag, causal, prefix_units):
    """What lies behind every sequence's end may hold anything, also where a prefix is said to be: it is NaN here."""
    new, lens, Hq, Hkv, D, page, prefix = case
    dt = {"bf16": torch.bfloat16, "f16": torch.float16}[tag]
    ops = _ops()
    k, v, table = make_cache([max(n, prefix) for n in lens], Hkv, D, page, dt, "hnd", 21, prefix)
    last = max(lens)                                       # positions [0, last) of the shared pages have been written
    for p in range(last, prefix // page * page):
        k[table[0, p // page], :, p % page] = v[table[0, p // page], :, p % page] = float("nan")
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    q = (torch.randn(cu[-1] + 2, Hq, D, generator=torch.Generator().manual_seed(5)) * 1.5).to(dt)
    told = [n if m else 250 for n, m in zip(lens, new)] if 0 in new and last == 60 else lens
    o, lse = ops.paged_gqa_fwd(q.cuda(), k.cuda(), v.cuda(), table.cuda(), _i32(told).cuda(), cu_q=_i32(cu).cuda(), shared_prefix=prefix, causal=causal)
    o64, lse64 = oracle.paged_attention(q, k, v, table, lens, cu, prefix, causal)
    assert within_weights(o, o64, q, k, v, table, lens, cu, prefix, causal)
    seen = torch.isfinite(lse64)
    assert torch.equal(torch.isfinite(lse.cpu()), seen) and (o.cpu()[~seen] == 0).all()
    assert ((lse.cpu().double() - lse64)[seen].abs() <= 2.0 ** -16 + 2.0 ** -23 * lse64[seen].abs()).all() and ops.kernel_status() == 0
