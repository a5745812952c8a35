"""DraftVerifier: the drafted-token operators run together, as a step that
verifies a tree, against the float64 restatement of the forward pass
(oracle/llama.py) and against the one-token decode step.

Tolerances are those of the decode step's tests, of the logits' scale: 2e-3
with fp32 activations and an fp16 cache; 6e-2 with Q8 activations or an int8
cache (a code is off by half a step, 1/254 of its row's largest value, as an
activation's is)."""
import dataclasses

import numpy as np
import pytest

from oracle.llama import LlamaRef
from test_gpu_decode import _oracle_weights, _tiny

pytestmark = pytest.mark.gpu


def model(act_mode, seed=7, head_dim=64):
    from odiengine_b200.decode import seeded_model

    cfg = dataclasses.replace(_tiny(act_mode), head_dim=head_dim)
    return cfg, seeded_model(cfg, seed=seed, interleave_gate_up=False)


def oracle_rows(ref, prefix, tokens, parents):
    """Each node's logits after prefix and its ancestors (one path at a time)."""
    paths = [[0]]
    for p in parents:
        paths.append(paths[p] + [len(paths)])
    rows = []
    for path in paths:
        for j, n in enumerate(path):
            lg = ref.step(tokens[n], len(prefix) + j)
        rows.append(lg)
    return np.stack(rows)


@pytest.mark.parametrize("act_mode,cache,tol", [(1, "f16", 2e-3), (1, "i8", 6e-2), (0, "f16", 6e-2), (0, "i8", 6e-2)])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_tree_logits_match_oracle(cuda_lib, act_mode, cache, tol, head_dim):
    from odiengine_b200.draft import DraftVerifier

    cfg, mw = model(act_mode, head_dim=head_dim)
    ref = LlamaRef(cfg, _oracle_weights(cuda_lib, cfg, mw))
    v = DraftVerifier(cfg, mw, cache=cache, max_nodes=12)
    prompt = [5, 17, 999, 3, 250, 8, 41, 700, 2, 90, 33, 61, 7, 500, 123]  # two chunks of the cache's rows
    v.start(prompt)
    for p, t in enumerate(prompt[:-1]):
        ref.step(t, p)
    assert v.pos == len(prompt) - 1
    drafted = [4, 9, 600, 31, 2, 77, 12, 300]
    parents = [0, 0, 1, 1, 2, 3, 6, 0]
    want = oracle_rows(ref, prompt[:-1], [prompt[-1]] + drafted, parents)
    kept_before = [c.k.clone() for c in v.caches]
    out = v.verify(drafted, parents)
    got = v.logits[:9].cpu().numpy().astype(np.float64)
    scale = np.abs(want).max()
    assert (np.abs(got - want) <= tol * scale).all(), np.abs(got - want).max() / scale
    assert out == [int(np.argmax(got[0]))] or len(out) > 1
    if cache == "f16":  # the prompt's rows are as they were
        for a, c in zip(kept_before, v.caches):
            assert (a[:, :len(prompt) - 1] == c.k[:, :len(prompt) - 1]).all()


@pytest.mark.parametrize("cache,head_dim", [("f16", 64), ("i8", 64), ("f16", 128), ("i8", 128)])
def test_drafts_do_not_change_what_is_generated(cuda_lib, cache, head_dim):
    """Good drafts, bad drafts, branches with the right token behind wrong
    ones: every call returns the tokens of undrafted greedy decoding, more at
    a time when the drafts were right; rows of the accepted path end up where
    undrafted decoding has them."""
    from odiengine_b200.draft import DraftVerifier, kv_read

    cfg, mw = model(1, head_dim=head_dim)
    prompt = [5, 17, 999, 3, 250]
    plain = DraftVerifier(cfg, mw, cache=cache)
    plain.start(prompt)
    want = []
    for _ in range(24):
        want += plain.verify()
    v = DraftVerifier(cfg, mw, cache=cache, max_nodes=32)
    v.start(prompt)
    got, calls, rng = [], 0, np.random.default_rng(0)
    while len(got) < 20:
        n = len(got)
        w = lambda i: want[n + i]  # noqa: E731
        bad = [int(t) for t in rng.integers(0, cfg.vocab, 6)]
        kind = calls % 4
        if kind == 0:    # a right chain of three
            out, least = v.verify([w(0), w(1), w(2)]), 4
        elif kind == 1:  # wrong first children, then the right one with a right child
            out, least = v.verify([(w(0) + 1) % cfg.vocab, (w(0) + 2) % cfg.vocab, w(0), bad[0], w(1)], [0, 0, 0, 1, 3]), 3
        elif kind == 2:  # nothing right
            out, least = v.verify([(w(0) + 1) % cfg.vocab, bad[1]]), 1
        else:            # right, then wrong
            out, least = v.verify([w(0), (w(1) + 1) % cfg.vocab]), 2
        assert len(out) >= least and out == want[n:n + len(out)], (kind, out, want[n:n + 6])
        got += out
        calls += 1
    assert v.pos == plain.pos - (len(want) - len(got)) and v.status() == 0
    n = v.pos
    for a, b in zip(v.caches, plain.caches):
        for x, y in zip(kv_read(a, 0, n), kv_read(b, 0, n)):
            # the same rows up to the rounding of T-token and one-token steps
            assert (x.float() - y.float()).abs().max() <= 2e-2 * y.float().abs().max()


def test_matches_the_decode_step(cuda_lib):
    """The verifier's tokens are those of DecodeModel's fused step wherever
    the top-2 gap exceeds the rounding of either."""
    from odiengine_b200.decode import DecodeModel
    from odiengine_b200.draft import DraftVerifier

    cfg, mw = model(1, seed=3)
    dm = DecodeModel(cfg, mw, mode="fused")
    prompt = [9, 1, 44, 723]
    dm.prefill(prompt[:-1])
    dm.reset(prompt[-1], len(prompt) - 1)
    v = DraftVerifier(cfg, mw)
    v.start(prompt)
    for _ in range(10):
        a, b = dm.generate(1), v.verify()
        la, lb = dm.logits.cpu().numpy(), v.logits[0].cpu().numpy()
        assert np.abs(la - lb).max() <= 4e-3 * np.abs(la).max()
        top = np.sort(la)[-2:]
        if top[1] - top[0] <= 8e-3 * np.abs(la).max():
            break
        assert a == b


@pytest.mark.parametrize("cache,head_dim", [("f16", 64), ("i8", 64), ("f16", 128), ("i8", 128)])
def test_steps_of_256_nodes(cuda_lib, cache, head_dim):
    """A prompt taken 256 tokens at a time, and a chain of 255 drafts, give what
    steps of 7 nodes give, within the roundings of the products' paths."""
    from odiengine_b200.decode import seeded_model
    from odiengine_b200.draft import DraftVerifier

    cfg = dataclasses.replace(_tiny(1), ctx=640, head_dim=head_dim)
    mw = seeded_model(cfg, seed=7, interleave_gate_up=False)
    rng = np.random.default_rng(4)
    prompt = [int(t) for t in rng.integers(0, cfg.vocab, 301)]
    wide, narrow = DraftVerifier(cfg, mw, cache=cache, max_nodes=256), DraftVerifier(cfg, mw, cache=cache, max_nodes=7)
    out = []
    for v in (wide, narrow):
        v.start(prompt)
        assert v.pos == 300
        out.append(v.verify())
    a, b = (v.logits[0].cpu().numpy() for v in (wide, narrow))
    assert np.abs(a - b).max() <= (4e-3 if cache == "f16" else 6e-2) * np.abs(b).max()
    drafted = [int(t) for t in rng.integers(0, cfg.vocab, 255)]
    wide.start(prompt)
    got = wide.verify(drafted)
    assert got[:1] == out[0] and wide.status() == 0
    a = wide.logits[200].cpu().numpy()  # the node after prompt + 200 drafts
    narrow.start(prompt + drafted[:200])
    narrow.verify()
    b = narrow.logits[0].cpu().numpy()
    assert np.abs(a - b).max() <= (4e-3 if cache == "f16" else 6e-2) * np.abs(b).max()


def test_penalties_masks_and_refusals(cuda_lib):
    import torch

    from odiengine_b200.draft import DraftVerifier

    cfg, mw = model(1)
    v = DraftVerifier(cfg, mw, max_nodes=8, history=16)
    with pytest.raises(RuntimeError):
        v.verify()
    v.start([5, 17, 999])
    first = v.verify()[0]
    lg = v.logits[0].clone()
    # banned, the token gives way to the next; a mask leaves one token
    v.start([5, 17, 999])
    second = v.verify(bias_ids=torch.tensor([first], dtype=torch.int32, device="cuda"),
                      bias=torch.tensor([-float("inf")], device="cuda"))[0]
    lg[first] = -float("inf")
    assert second == int(lg.argmax()) != first
    mask = torch.zeros((1, (cfg.vocab + 31) // 32), dtype=torch.int32, device="cuda")
    mask[0, 3] = 1 << 5
    v.start([5, 17, 999])
    assert v.verify(mask=mask) == [101]
    mask.zero_()
    v.start([5, 17, 999])
    with pytest.raises(RuntimeError):
        v.verify(mask=mask)
    v.start([5, 17, 999])
    v.verify([first], repeat_penalty=1.5, presence_penalty=0.5)  # node 1 counts its ancestor too
    for bad in (dict(drafted=[1] * 8), dict(drafted=[1], parents=[1]), dict(drafted=[cfg.vocab]), dict(drafted=[1, 2], parents=[0])):
        with pytest.raises(ValueError):
            v.verify(**bad)
    with pytest.raises(ValueError):
        v.start([])
    with pytest.raises(ValueError):
        v.start(list(range(cfg.ctx + 1)))
    v.start(list(range(cfg.ctx)))
    assert len(v.verify()) == 1  # the context's last slot
    with pytest.raises(ValueError):
        v.verify()
    plain = DraftVerifier(cfg, mw, device="cuda")
    plain.start([5, 17, 999])
    with pytest.raises(ValueError):  # nothing that it could count
        plain.verify(repeat_penalty=1.5)
    from odiengine_b200.decode import seeded_model
    with pytest.raises(ValueError):
        DraftVerifier(cfg, seeded_model(cfg, interleave_gate_up=True))


def test_verifiers_keep_their_workspaces(cuda_lib):
    """Two verifiers and a DecodeModel over the same weights: building one
    leaves the others' workspaces alone, and steps that run at the same time on
    two streams give what they give one after the other."""
    import threading

    import torch

    from odiengine_b200.decode import DecodeModel
    from odiengine_b200.draft import DraftVerifier

    cfg, mw = model(0)  # Q8: a product of several tokens quantises them into its workspace
    dm = DecodeModel(cfg, mw, mode="fused")
    held = [dw._ws for lw in mw.layers for dw in (lw.wqkv, lw.wo, lw.wgu, lw.wdown)] + [mw.output._ws]
    vs = [DraftVerifier(cfg, mw, max_nodes=n) for n in (8, 32)]
    now = [dw._ws for lw in mw.layers for dw in (lw.wqkv, lw.wo, lw.wgu, lw.wdown)] + [mw.output._ws]
    assert all(a is b for a, b in zip(held, now)) and dm.status() == 0
    rng = np.random.default_rng(12)
    nodes = [[int(t) for t in rng.integers(0, cfg.vocab, n)] for n in (8, 32)]
    for v, n in zip(vs, nodes):
        v.start([5, 17, n[0]])
    want, streams = [], [torch.cuda.Stream() for _ in vs]
    for v, n in zip(vs, nodes):
        v._forward(n, None, None, True)
        want.append(v.logits[:len(n)].clone())
    torch.cuda.synchronize()
    wrong = [0, 0]

    def run(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(60):
                vs[i]._forward(nodes[i], None, None, True)
                wrong[i] += not torch.equal(vs[i].logits[:len(nodes[i])], want[i])

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert wrong == [0, 0] and all(v.status() == 0 for v in vs)


@pytest.mark.parametrize("cache", ["f16", "i8"])
def test_calls_on_other_streams_follow_each_other(cuda_lib, cache):
    """A verifier made on one stream (whose fills come late) and called on others
    (where a branch's rows come late into place) gives what it gives on one."""
    import torch

    from odiengine_b200.draft import DraftVerifier

    cfg, mw = model(1)
    prompt = [5, 17, 999, 3, 250]
    plain = DraftVerifier(cfg, mw, cache=cache)
    plain.start(prompt)
    want = []
    for _ in range(6):
        want += plain.verify()
    drafts = [(want[0] + 1) % cfg.vocab, want[0], want[1]]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda._sleep(100_000_000)
    v = DraftVerifier(cfg, mw, cache=cache, max_nodes=8)
    with torch.cuda.stream(streams[0]):
        v.start(prompt)
    with torch.cuda.stream(streams[1]):
        first = v.verify(drafts, [0, 0, 2])  # the second branch is right: its rows move
        torch.cuda._sleep(100_000_000)
    with torch.cuda.stream(streams[2]):
        second = v.verify()
    torch.cuda.synchronize()
    assert first == want[:3] and second == want[3:4]
