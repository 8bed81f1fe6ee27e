"""PairDropout's masks over blocks, updates and steps: no two draw from the same
place of the generator, whatever a caller adds to ``step`` between replays."""

from __future__ import annotations

import dataclasses

import pytest
import torch

from foldjax_amd import kernels, openfold3
from foldjax_amd import pairformer as PF
from foldjax_amd.pairformer import PairDropout, PairformerLayerWeights, TriangleSublayers
from tests.gpu_util import say


@pytest.fixture
def places(monkeypatch):
    """Where each call of dropout_add draws: offset + step, as the kernel adds them."""
    seen = []

    def drop(x, *, seed, offset, step, **_):
        assert 0 <= seed < 2**64 and 0 <= offset < 2**64
        seen.append((offset + (0 if step is None else int(step))) % 2**64)
        return x

    update = lambda z, *a, residual=None, **k: z.clone()  # noqa: E731
    for name in ("trimul", "triattn"):
        monkeypatch.setattr(kernels, name, update)
    for name in ("triangle_multiplication", "triangle_attention"):
        monkeypatch.setattr(openfold3, name, update)
    monkeypatch.setattr(openfold3, "swiglu_transition", update)
    monkeypatch.setattr(kernels, "dropout_add", drop)
    return seen


def block(z, dropout):
    TriangleSublayers(None, None, None, None).forward(z, None, dropout=dropout)


def of3_block(z, dropout):
    params = openfold3.PairBlockParams(None, None, None, None, None)
    openfold3.pair_block(z, params, pair_mask=None, no_heads_pair=4, dropout=dropout)


@pytest.mark.parametrize("offset", [0, 11, 2**64 - 3 * 2**32 - 5])
@pytest.mark.parametrize("stride", [1, 2, 3, 4, 8, 100])
@pytest.mark.parametrize("run", [block, of3_block], ids=["block", "openfold3"])
def test_no_place_is_drawn_from_twice(places, run, stride, offset):
    step = torch.zeros((), dtype=torch.int64)
    drop = PairDropout(seed=7, offset=offset, step=step)
    z = torch.zeros(1, 2, 2, 8)
    for _ in range(40):
        for layer in range(3):
            run(z, PF._block_dropout(drop, layer))
        step += stride
    assert len(places) == 40 * 3 * 4
    assert len(set(places)) == len(places)


def test_a_step_of_four_is_four_offsets_and_no_step_is_zero(places):
    """A block's updates draw at offset .. offset + 3, and 4 k further on at step 4 k."""
    z = torch.zeros(1, 2, 2, 8)
    block(z, PairDropout(offset=9))
    block(z, PairDropout(offset=9, step=torch.tensor(0)))
    block(z, PairDropout(offset=1, step=torch.tensor([8])))
    assert places == [9, 10, 11, 12] * 3


@pytest.mark.parametrize("more", [{"offset": -1}, {"offset": 2**64}, {"seed": -1}, {"seed": 2**64}], ids=str)
def test_places_out_of_range_are_refused(more):
    with pytest.raises(ValueError, match="seed and offset"):
        PairDropout(**more)


@pytest.mark.gpu
def test_a_captured_stack_stepping_by_one_never_repeats_a_mask():
    say("captured stack dropout by one")
    bf = torch.bfloat16
    blocks = [PairformerLayerWeights.random(bf, "cuda", seed=s).triangle for s in (3, 5)]
    g = torch.Generator().manual_seed(0)
    z = torch.randn(1, 16, 16, 128, generator=g).to(bf).cuda()
    step = torch.zeros((), dtype=torch.int64, device="cuda")
    drop = PairDropout(p=0.25, seed=1, offset=8, step=step)

    def stack(dropout):
        x = z
        for i, b in enumerate(blocks):
            x = b.forward(x, None, dropout=dropout.of_block(i))
        return x

    stack(drop)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = stack(drop)
        step += 1
    outs = []
    for i in range(6):
        graph.replay()
        torch.cuda.synchronize()
        outs.append(got.clone())
        assert torch.equal(got, stack(dataclasses.replace(drop, step=torch.tensor(i, device="cuda")))), f"replay {i}"
    # the masks themselves, of the updates of one shape
    ones = torch.ones(1, 16, 16, 128, dtype=bf, device="cuda")
    masks = []
    for i in range(6):
        for b in range(2):
            d = dataclasses.replace(drop, step=torch.tensor(i, device="cuda")).of_block(b).drawn()
            masks += [d.add(ones.clone(), torch.zeros_like(ones), s, False, None, None) for s in range(4)]
    for i, a in enumerate(masks):
        assert not any(torch.equal(a, b) for b in masks[:i]), i
    assert not any(torch.equal(a, b) for i, a in enumerate(outs) for b in outs[:i])
