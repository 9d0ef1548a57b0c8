"""The sparse layer of examples/sparse_decode.py: prompt chunks, then decode steps."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from dsa_b200.build import build

    build()
    path = Path(__file__).resolve().parents[1] / "examples" / "sparse_decode.py"
    spec = importlib.util.spec_from_file_location("sparse_decode", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("batch,prompt,chunk,steps", [(1, 100, 33, 3), (3, 301, 128, 4)])
def test_a_top_k_of_every_position_is_dense_attention(example, batch, prompt, chunk, steps):
    r = example.run(batch, prompt, chunk, steps, topk=4096)
    # both round their weights and outputs to bfloat16 (2^-8 each, of sums over many keys)
    assert r["sparse_vs_dense"] < 2.0 ** -7


def test_chunks_do_not_change_the_prompt(example):
    # whole or in pieces: the same positions, the same rotation, the same attention
    outs = []
    for pieces in ([257], [100, 1, 156], [1] * 3 + [254]):
        layer = example.SparseLayer(2, 260, topk=64)
        x = torch.randn(2, 257, 2048, generator=torch.Generator().manual_seed(3))
        x = x.to(torch.bfloat16).cuda()
        at, got = 0, []
        for n in pieces:
            got.append(layer.chunk(x[:, at:at + n]))
            at += n
        outs.append(torch.cat(got, 1).double())
    for other in outs[1:]:
        err = (other - outs[0]).norm() / outs[0].norm()
        # the projection's bfloat16 rounding may fall differently for other batch sizes
        assert float(err) < 2.0 ** -6


def test_a_small_top_k_attends_to_the_selected_positions_only(example):
    layer = example.SparseLayer(2, 520, topk=32)
    g = torch.Generator().manual_seed(4)
    layer.chunk(torch.randn(2, 500, 2048, generator=g).to(torch.bfloat16).cuda())
    x = torch.randn(2, 2048, generator=g).to(torch.bfloat16).cuda()
    out = layer.step(x)
    iq, iw = layer.projector.q, layer.projector.w
    from dsa_b200 import scores_topk

    idx, _ = scores_topk(iq, iw, layer.index_keys[:, :501], 32, sorted=False)
    q = layer._qkv(x)[0]
    q = layer.appender.append(layer.step_batch, *layer._qkv(x)[1:], q)
    for b in range(2):
        flat = layer.cache.keys[layer.table[b].long()].flatten(0, 1)[idx[b].long()].double()
        vals = layer.cache.values[layer.table[b].long()].flatten(0, 1)[idx[b].long()].double()
        z = torch.einsum("hgd,khd->hgk", q[b].double().view(4, 4, 128), flat) / 128 ** 0.5
        w = torch.softmax(z, -1)
        want = torch.einsum("hgk,khd->hgd", w, vals).reshape(16, 128)
        size = torch.einsum("hgk,khd->hgd", w, vals.abs()).reshape(16, 128)
        u = 2.0 ** -8
        err = (out[b].double() - want).abs()
        assert bool((err <= (u + 2.0 ** -12) * size + u * (1 + u) * want.abs()).all())
