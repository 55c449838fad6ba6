"""GPU: the examples of the verify step of many requests, in the project's pages of text and in its module, run as they
stand where one of the requests has no room."""
import glob
import os
import re

import pytest
import torch

import momij_amd.paged
import paged_ref as R
from test_gpu_paged_attn import D, cfg, ctx, cuda  # noqa: F401

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NQ, NKV, LAYERS, V, N, STEPS = 16, 4, 3, 500, 3, 4


def examples():
    for page in sorted(glob.glob(os.path.join(ROOT, "*.md"))):
        for code in re.findall(r"```python\n(.*?)```", open(page).read(), re.S):
            if "pages_reserve" in code:
                yield pytest.param(code, STEPS, id=os.path.basename(page))
    code = re.search(r"\n\n((?:    [^\n]*\n)+)", momij_amd.paged.__doc__).group(1)
    yield pytest.param("from momij_amd.paged import PagedCache, RowBatch\n" + re.sub(r"(?m)^    ", "", code), 1,
                       id="paged.py")


@pytest.mark.parametrize("code,count", list(examples()))
@pytest.mark.parametrize("tree", [False, True])
def test_a_request_without_room(ctx, code, count, tree):  # noqa: F811
    """Three requests of three rows a step and pages for two: these go on, the third stays where it was."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(3)
    rows = 3 * N
    qkv = [torch.randn((rows, (NQ + 2 * NKV) * D), generator=gen, device="cuda").half() for _ in range(LAYERS)]
    logits = torch.randn((rows, V), generator=gen, device="cuda")
    out = torch.zeros((rows, NQ * D), dtype=torch.float16, device="cuda")
    one = torch.ones(D, dtype=torch.float16, device="cuda")
    tokens = torch.randint(0, V, (rows,), generator=gen, device="cuda").int()
    uniforms = torch.zeros(rows, device="cuda"), torch.rand(N, generator=gen, device="cuda")  # (all drafts are accepted)

    names = dict(
        ctx=ctx, n_seqs=N, n_pages=2, n_kv_heads=NKV, blocks=4, n_layers=LAYERS, n_heads=NQ, window=0, cfg=cfg(NQ, NKV, 64),
        row_start=cuda([0, 3, 6, 9]), rows=rows, max_rows=3,
        anc=cuda(momij_amd.paged.tree_masks([-1, 0, 0]) * N, torch.int64) if tree else None, reserved=cuda([[5] * 4] * N),
        qkv=qkv[0], project=lambda layer, tokens: qkv[layer], head=lambda out: logits, q_norm_w=one, k_norm_w=one,
        q=torch.zeros_like(out), out=out, logits=logits, tokens=tokens, temperature=torch.ones(N, device="cuda"),
        u_accept=uniforms[0], u_sample=uniforms[1], steps=[(tokens, *uniforms)] * STEPS, accepted=cuda([0] * N),
        path=cuda([0] * rows), token=cuda([0] * N), lengths=cuda([-1] * N), source=cuda([-1] * N))
    exec(compile(code, "example", "exec"), names)
    ctx.sync()
    cache, kept = names["cache"], 2 if tree else 3  # (the second of two siblings is not reached)
    assert names["reserved"][:, 0].tolist() == [1, 1, 0]
    assert cache.lens.tolist() == [kept * count, kept * count, 0]
    assert (cache.table >= 0).sum(1).tolist() == [1, 1, 0] and cache.refs.tolist() == [1, 1]
    several = "project" in code
    for l in range(LAYERS):
        for s in range(2):
            v = R.rows_of(cache, l, s, torch.arange(kept * count, device="cuda"))[1]
            x = qkv[l if several else 0].reshape(rows, -1, D)[3 * s:3 * s + kept, NQ + NKV:].double()
            assert torch.equal(v, x.repeat(count, 1, 1))
