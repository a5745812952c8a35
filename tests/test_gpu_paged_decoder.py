"""PagedDecoder: the operators over a paged cache run together, for several
requests, against the float64 restatement of the forward pass (oracle/llama.py)
and, for what is chosen, against the plain rule on the decoder's own logits.

Tolerances, of the logits' scale: 2e-3 is what the decode step's tests allow with
fp32 activations and an fp16 cache.  Here q, the weights of the softmax and the
cached rows are rounded, each by half a step: fp16 adds twice 2^-11 to that, and
bf16's half step is 2^-8 for each of the three."""
import dataclasses

import numpy as np
import pytest
import torch

import paged_ref
from oracle.llama import LlamaRef
from test_gpu_decode import _oracle_weights, _tiny

pytestmark = pytest.mark.gpu
TOL = {torch.float16: 2e-3 + 2 * 2.0 ** -11, torch.bfloat16: 2e-3 + 3 * 2.0 ** -8}


def model(head_dim=64, seed=7, ctx=64):
    from odiengine_b200.decode import seeded_model

    cfg = dataclasses.replace(_tiny(1), head_dim=head_dim, ctx=ctx)
    return cfg, seeded_model(cfg, seed=seed, interleave_gate_up=False)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("head_dim,page_size,chunk", [(64, 16, 5), (128, 32, 40)])
def test_logits_match_the_oracle(cuda_lib, dtype, head_dim, page_size, chunk):
    """Requests that come and go, prompts in chunks beside decoding requests, drafts
    that are refused: every row of logits is that of its own sequence."""
    from odiengine_b200.paged import PagedDecoder

    cfg, mw = model(head_dim)
    W = _oracle_weights(cuda_lib, cfg, mw)
    d = PagedDecoder(cfg, mw, requests=3, num_pages=3 * 64 // page_size, page_size=page_size, dtype=dtype, max_drafts=3, chunk=chunk)
    rng = np.random.default_rng(0)
    prompts = [rng.integers(0, cfg.vocab, n).tolist() for n in (1, 23, 9)]
    seqs = {}
    for p in prompts:
        b = d.add(p)
        seqs[b] = {"ref": LlamaRef(cfg, W), "tokens": p[:-1], "fed": 0, "pending": p[-1]}
    steps, swapped = 0, False
    while steps < 8:
        ready = [b for b in sorted(seqs) if not d.left(b)]
        drafts = {b: rng.integers(0, cfg.vocab, int(rng.integers(0, 4))).tolist() for b in ready}
        before = {b: d.left(b) for b in seqs}
        out = d.step(drafts)
        row = 0
        for b in sorted(seqs):
            s = seqs[b]
            if before[b]:
                continue
            for i in range(s["fed"], len(s["tokens"])):
                s["ref"].step(s["tokens"][i], i)
            s["fed"] = len(s["tokens"])
            fed = [s["pending"], *drafts.get(b, ())]
            want = np.stack([s["ref"].step(t, len(s["tokens"]) + i) for i, t in enumerate(fed)])
            got = d.logits[row:row + len(fed)].cpu().numpy().astype(np.float64)
            row += len(fed)
            assert np.abs(got - want).max() <= TOL[dtype] * np.abs(want).max(), np.abs(got - want).max() / np.abs(want).max()
            greedy = got.argmax(1).tolist()
            kept = 0
            while kept + 1 < len(fed) and fed[kept + 1] == greedy[kept]:
                kept += 1
            assert out[b] == [*fed[1:1 + kept], greedy[kept]]
            s["tokens"] += fed[:1 + kept]
            s["fed"] = len(s["tokens"])
            s["pending"] = out[b][-1]
        steps += bool(ready)
        if steps == 4 and not swapped:  # one leaves, another comes in its place
            swapped = True
            d.finish(0)
            del seqs[0]
            p = rng.integers(0, cfg.vocab, 17).tolist()
            assert d.add(p) == 0
            seqs[0] = {"ref": LlamaRef(cfg, W), "tokens": p[:-1], "fed": 0, "pending": p[-1]}
    assert d.status() == 0
    held = sum(-(-n // page_size) for n in d._len)
    assert d.free_pages == d.num_pages - held


def test_good_drafts_are_kept(cuda_lib):
    """What a request generates one token at a time is kept when it is drafted to
    another request of the same prompt, and both go on alike."""
    from odiengine_b200.paged import PagedDecoder

    cfg, mw = model(seed=3)
    d = PagedDecoder(cfg, mw, requests=2, num_pages=16, max_drafts=4)
    a = d.add([5, 17, 999, 3, 250])
    while d.left(a):
        d.step()
    text = [d.step()[a][0] for _ in range(9)]
    b = d.add([5, 17, 999, 3, 250])
    while d.left(b):
        text += d.step().get(a, [])
    got = d.step({b: text[:4]})[b]
    assert got == text[:5]
    assert d.step({b: [text[5], (text[6] + 1) % cfg.vocab, text[7]]})[b] == text[5:7]


@pytest.mark.parametrize("temperature", [0.7, 1.3])
def test_sampling_follows_the_rule(cuda_lib, temperature):
    from odiengine_b200.paged import PagedDecoder

    cfg, mw = model()
    g = torch.Generator(device="cuda").manual_seed(5)
    d = PagedDecoder(cfg, mw, requests=3, num_pages=24, max_drafts=5, temperature=temperature, generator=g)
    ids = [d.add([1 + i, 50, 600]) for i in range(3)]
    while any(d.left(b) for b in ids):
        d.step()
    d.step()
    for _ in range(4):
        fed, drafts = {}, {}
        for b in ids:  # what the target thinks likely of the pending row, then anything
            drafts[b] = [int(d.logits[b % 3].argmax())] + [7, 8][:b]
            fed[b] = [d._todo[b][0], *drafts[b]]
        out = d.step(drafts)
        rows = [t for b in ids for t in fed[b]]
        starts = np.concatenate([[0], np.cumsum([len(fed[b]) for b in ids])]).tolist()
        acc, nxt = paged_ref.verify(d.logits[:len(rows)].cpu().numpy(), rows, starts, d.u_accept.tolist(), d.u_next.tolist(), temperature)
        for i, b in enumerate(ids):
            assert out[b] == [*drafts[b][:acc[i]], nxt[i]]


def test_what_a_decoder_refuses(cuda_lib):
    from odiengine_b200.paged import PagedDecoder

    cfg, mw = model()
    d = PagedDecoder(cfg, mw, requests=2, num_pages=3, max_drafts=2, chunk=16)
    for bad in ([], [cfg.vocab], [1] * (cfg.ctx + 1)):
        with pytest.raises(ValueError):
            d.add(bad)
    with pytest.raises(ValueError):
        d.finish(0)
    a = d.add(list(range(33)))
    with pytest.raises(ValueError):  # its prompt first
        d.step({a: [1]})
    while d.left(a):
        d.step()
    b = d.add([1] * 20)
    with pytest.raises(RuntimeError):  # two pages each, three there are
        while True:
            d.step()
    for drafts in ({a: [1, 2, 3]}, {a: [-1]}, {7: [1]}):
        with pytest.raises(ValueError):
            d.step(drafts)
    with pytest.raises(RuntimeError):
        d.add([1])
    d.finish(a)
    while d.left(b):
        d.step()
    assert len(d.step()[b]) == 1 and d.status() == 0
    for kw in (dict(temperature=0.0), dict(max_drafts=-1), dict(chunk=0)):
        with pytest.raises(ValueError):
            PagedDecoder(cfg, mw, requests=2, num_pages=3, **kw)
