"""GPU: the checked build of the library on the serving operators' other routes.

Held against its extent is, before the access, every element of the block table, the lengths and offsets, q, o, lse, the
caches, the workspace's partials, the projections, angles and positions, and every row of a sampling call; what a TMA box
covers is held by its tensor map.  Status 7 otherwise: these calls leave 0 and give the default build's results."""
import json
import os
import subprocess
import sys

import pytest

from test_gpu_serving_boundary import CHECKED, ROOT

pytestmark = pytest.mark.gpu

CHILD = r"""
import hashlib, json, os, sys, torch
sys.path.insert(0, os.environ["ARKE_ROOT"])
from arke_b200 import ops, _lib
out = {"version": _lib.version()}
def h(*ts):
    m = hashlib.sha256()
    for t in ts:
        m.update(t.detach().contiguous().cpu().reshape(-1).view(torch.uint8).numpy().tobytes())
    return m.hexdigest()
g = torch.Generator(device="cuda").manual_seed(0)
i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
CASES = [  # new, lens, Hq, Hkv, D, page, shared prefix, longest told
    ([0] * 40 + [90] + [0] * 50, [5] * 40 + [140] + [3] * 50, 8, 2, 64, 16, 0, 90),
    ([0] * 40 + [90] + [0] * 50, [5] * 40 + [140] + [3] * 50, 8, 2, 64, 16, 0, 0),
    ([1] * 24, [1100 + 40 * i for i in range(24)], 8, 2, 128, 32, 1024, 0),
    ([1] * 3, [97, 130, 100], 4, 2, 64, 16, 96, 0),
    ([20, 1, 9], [300, 200, 700], 7, 1, 64, 8, 150, 20),
    ([300], [2000], 4, 2, 128, 16, 0, 300),
    ([2] * 200, [30 + b for b in range(200)], 4, 4, 64, 4, 0, 0),
    ([1, 1], [0, 0], 2, 1, 64, 16, 0, 0)]
for n, (new, lens, Hq, Hkv, D, page, prefix, longest) in enumerate(CASES):
    pages = [-(-x // page) for x in lens]
    k, v = (torch.randn(sum(pages) + 1, Hkv, page, D, generator=g, device="cuda").half() for _ in range(2))
    table, at = torch.full((len(new), max(pages) + 2), 1 << 30, dtype=torch.int32), 0
    for b, m in enumerate(pages):
        table[b, :m] = torch.arange(at, at + m)
        at += m
    cu = [0]
    for x in new:
        cu.append(cu[-1] + x)
    table, L, cu_q, T = table.cuda()[:, :max(pages) + 1], i32(lens), i32(cu), cu[-1] + 2
    wide = torch.randn(T, (Hq + 2 * Hkv) * D, generator=g, device="cuda").half()
    cos, sin = (torch.rand(max(lens) + 50, D // 2, generator=g, device="cuda") for _ in range(2))
    pos = torch.randint(max(lens) + 50, (T,), generator=g, device="cuda").int()
    q = ops.qkv_rope_paged_append(wide, cos, sin, k, v, table, L, Hq, cu_q=cu_q, positions=pos)
    if min(l - x for l, x in zip(lens, new)) < 0:
        ops.kernel_status()                       # tokens in front of their sequence: reported, not stored
    out[f"append{n}"] = h(q, k, v)
    packed = wide.view(T, Hq + 2 * Hkv, D)[:, :Hq]
    heads = q.transpose(0, 1).contiguous().transpose(0, 1)
    for name, x in (("packed", packed), ("heads", heads), ("one token", q[:1].expand(T, Hq, D))):
        for kb in (1, 1 << 30):
            with ops.options(paged_prefix_kb=kb):
                out[f"attend{n}{name}{kb}"] = h(*ops.paged_gqa_fwd(x, k, v, table, L, cu_q=cu_q, shared_prefix=prefix, max_new=longest))
for n, (B, V, dt) in enumerate([(3, 128256, torch.float32), (300, 4099, torch.bfloat16), (2, 1 << 20, torch.float32)]):
    x = (torch.randn(B, V, generator=g, device="cuda") * 0.01 - 29).to(dt)
    x[:, -1] = 0
    u = torch.linspace(0, 1, B, device="cuda")
    for f in (dict(), dict(top_p=1 - 2.0 ** -24), dict(top_k=V // 2, top_p=1 - 2.0 ** -23), dict(min_p=1e-20)):
        out[f"sample{n}{f}"] = h(*ops.sample_tokens(x, u, return_logprob=True, **f))
torch.cuda.synchronize()
out["status"] = ops.kernel_status()
print("RESULT " + json.dumps(out))
"""


def _run(lib):
    env = dict(os.environ, ARKE_ROOT=str(ROOT))
    env.pop("ARKE_B200_SO", None)
    if lib is not None:
        env["ARKE_B200_SO"] = str(lib)
    p = subprocess.run([sys.executable, "-c", CHILD], env=env, capture_output=True, text=True, timeout=900)
    assert p.returncode == 0, p.stderr[-3000:]
    return json.loads([ln for ln in p.stdout.splitlines() if ln.startswith("RESULT ")][-1][len("RESULT "):])


def test_checked_build_of_the_other_routes():
    if not CHECKED.exists():
        pytest.skip("checked library not built (python -m arke_b200.build --flag=-DARKE_B200_CHECKED --out ...)")
    checked, default = _run(CHECKED), _run(None)
    assert "checked build" in checked.pop("version") and "checked build" not in default.pop("version")
    assert checked["status"] == 0 and default["status"] == 0
    assert [k for k in default if default[k] != checked[k]] == [] and len(default) >= 60
