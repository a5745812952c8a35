"""PagedDecoder: which batch a step runs in, and the options that a model may have."""
import dataclasses

import numpy as np
import pytest
import torch

import paged_ref
from oracle.llama import LlamaRef
from test_gpu_decode import _oracle_weights, _tiny
from test_gpu_paged_decoder import TOL

pytestmark = pytest.mark.gpu


def model(seed=7, **kw):
    from odiengine_b200.decode import seeded_model

    cfg = dataclasses.replace(_tiny(1), **kw)
    return cfg, seeded_model(cfg, seed=seed, interleave_gate_up=False)


@pytest.mark.parametrize("temperature", [None, 0.9])
@pytest.mark.parametrize("max_drafts", [7, 0])
def test_single_tokens_run_in_a_batch_of_single_tokens(cuda_lib, monkeypatch, temperature, max_drafts):
    """The batch's max_new chooses attention's kernel: one of drafts for single tokens of
    eight heads per kv head would be one for 64 rows with 8 in use.  Whatever the
    batch, a request's logits are those of its own sequence."""
    from odiengine_b200 import paged

    cfg, mw = model(heads=8, kv_heads=1)
    W = _oracle_weights(cuda_lib, cfg, mw)
    used = []
    real = paged.attention_paged
    monkeypatch.setattr(paged, "attention_paged", lambda q, c, t, b, *a, **kw: (used.append(b.max_new), real(q, c, t, b, *a, **kw))[1])
    g = torch.Generator(device="cuda").manual_seed(1)
    d = paged.PagedDecoder(cfg, mw, requests=3, num_pages=12, max_drafts=max_drafts, chunk=6, temperature=temperature, generator=g)
    ids = [d.add(p) for p in ([3, 4, 5], [9], [7, 8])]
    d.step()
    assert set(used) == {6, 1}  # two prompts in a chunk, the other's first token
    while any(d.left(b) for b in ids):
        d.step()
    refs = {b: (LlamaRef(cfg, W), []) for b in ids}
    fed = {0: [3, 4], 1: [9], 2: [7]}
    for b in ids:  # what is in the cache so far
        ref, toks = refs[b]
        assert d._len[b] == len(fed[b])
        for i, t in enumerate(fed[b]):
            ref.step(t, i)
        toks += fed[b]
    for drafts in ({}, {0: [1, 2], 2: [5]}, {}, {1: [6] * 7}, {}):
        drafts = {b: x[:max_drafts] for b, x in drafts.items()}
        used.clear()
        pending = {b: d._todo[b][0] for b in ids}
        out = d.step(drafts)
        assert set(used) == {1 + max_drafts if any(drafts.values()) else 1}
        lists, row, starts = {}, 0, [0]
        for b in ids:
            ref, toks = refs[b]
            lists[b] = [pending[b], *drafts.get(b, ())]
            want = np.stack([ref.step(t, len(toks) + i) for i, t in enumerate(lists[b])])
            got = d.logits[row:row + len(want)].cpu().numpy().astype(np.float64)
            assert np.abs(got - want).max() <= TOL[torch.float16] * np.abs(want).max()
            row += len(want)
            starts.append(row)
        logits, rows = d.logits[:row].cpu().numpy(), [t for b in ids for t in lists[b]]
        if temperature:
            acc, nxt = paged_ref.verify(logits, rows, starts, d.u_accept.tolist(), d.u_next.tolist(), temperature)
        for i, b in enumerate(ids):
            if not temperature:
                best = logits[starts[i]:starts[i + 1]].argmax(1)
                kept = next(k for k in range(len(best)) if k + 1 == len(best) or best[k] != lists[b][k + 1])
                assert out[b] == [*lists[b][1:1 + kept], best[kept]]
            else:
                assert out[b] == [*lists[b][1:1 + acc[i]], nxt[i]]
            refs[b][1].extend(lists[b][:len(out[b])])
    assert d.status() == 0
